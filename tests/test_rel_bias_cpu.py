"""Host-side behaviour of window attention with a relative position bias: bucket indexes, refusals."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import flash_aurora_b200 as fa


def test_window_buckets_are_swin_offsets():
    b = fa.RelativeBuckets.window((2, 3, 4))
    assert b.tokens == 24 and b.num_buckets == 3 * 5 * 7
    coords = [(c, h, w) for c in range(2) for h in range(3) for w in range(4)]
    for i, a in enumerate(coords):
        for j, c in enumerate(coords):
            d = [x - y for x, y in zip(a, c)]
            assert int(b.index[i, j]) == ((d[0] + 1) * 5 + d[1] + 2) * 7 + d[2] + 3


def test_log_distance_buckets():
    b = fa.RelativeBuckets.log_distance(140, num_buckets=32, max_distance=128)
    idx = b.index
    for i, j in ((0, 0), (5, 0), (0, 7), (20, 12), (139, 0), (0, 139), (3, 60)):
        d = abs(j - i)
        far = 8 + int(math.log(max(d, 1) / 8) / math.log(16) * 8) if d >= 8 else 0
        assert int(idx[i, j]) == (16 if j > i else 0) + (d if d < 8 else min(far, 15))
    assert int(idx.min()) == 0 and int(idx.max()) < 32


def test_bucket_lists_cover_every_pair():
    g = torch.Generator().manual_seed(0)
    index = torch.randint(0, 9, (13, 13), generator=g)
    b = fa.RelativeBuckets(index, 11)
    assert sorted(b.order.tolist()) == list(range(169))
    for n in range(11):
        members = b.order[int(b.offsets[n]):int(b.offsets[n + 1])].long()
        assert torch.equal(members, (index.reshape(-1) == n).nonzero().reshape(-1))
    index.fill_(0)
    assert int(b.index.max()) > 0  # the index is a copy


@pytest.mark.parametrize("index,nb,match", [
    (torch.zeros(3, 4, dtype=torch.long), 2, r"\(N, N\)"),
    (torch.zeros(145, 145, dtype=torch.long), 2, "144"),
    (torch.zeros(0, 0, dtype=torch.long), 2, "144"),
    (torch.zeros(3, 3), 2, "integers"),
    (torch.full((3, 3), 2), 2, "outside"),
    (torch.full((3, 3), -1), 2, "outside"),
    (torch.zeros(3, 3, dtype=torch.long), 0, "positive"),
])
def test_bucket_refusals(index, nb, match):
    with pytest.raises(ValueError, match=match):
        fa.RelativeBuckets(index, nb)


def test_bucket_constructor_refusals():
    with pytest.raises(ValueError, match="three positive"):
        fa.RelativeBuckets.window((2, 6))
    with pytest.raises(ValueError, match="three positive"):
        fa.RelativeBuckets.window((2, 0, 6))
    with pytest.raises(ValueError, match="multiple of 4"):
        fa.RelativeBuckets.log_distance(16, num_buckets=6)
    with pytest.raises(ValueError, match="max_distance"):
        fa.RelativeBuckets.log_distance(16, num_buckets=32, max_distance=8)


def test_attention_refusals_before_any_launch():
    b = fa.RelativeBuckets.window((1, 2, 4))
    t = torch.zeros(b.num_buckets, 2)
    q = torch.zeros(3, 2, 8, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        fa.window_attn_rel_bias(q, q, q, t, b)
    with pytest.raises(RuntimeError, match="CUDA"):
        fa.window_attn_rel_bias_qkvpacked(torch.zeros(3, 8, 384), 2, t, b)
    with pytest.raises(TypeError, match="bfloat16 and float32"):
        fa.window_attn_rel_bias(q.half(), q.half(), q.half(), t, b)
    with pytest.raises(ValueError, match="share a dtype"):
        fa.window_attn_rel_bias(q, q.bfloat16(), q, t, b)
    with pytest.raises(ValueError, match=r"\(Bwin, H, N, Dh\)"):
        fa.window_attn_rel_bias(q, q[:, :1], q, t, b)
    with pytest.raises(ValueError, match="head_dim 64"):
        fa.window_attn_rel_bias(q[..., :32], q[..., :32], q[..., :32], t, b)
    with pytest.raises(ValueError, match="1 to 144"):
        big = torch.zeros(1, 1, 145, 64)
        fa.window_attn_rel_bias(big, big, big, t, b)
    with pytest.raises(ValueError, match="output_layout"):
        fa.window_attn_rel_bias_qkvpacked(torch.zeros(3, 8, 384), 2, t, b, output_layout="nhd")
    with pytest.raises(ValueError, match="divisible"):
        fa.window_attn_rel_bias_qkvpacked(torch.zeros(3, 8, 380), 2, t, b)
    with pytest.raises(ValueError, match="contiguous"):
        fa.window_attn_rel_bias_qkvpacked(torch.zeros(3, 8, 768)[..., :384], 2, t, b)


def test_abi_refusals_without_a_gpu():
    from flash_aurora_b200 import _lib
    lib = _lib.load()
    p = ctypes.c_void_p(1 << 20)
    st = (ctypes.c_int64 * 21)(*([64] * 21))

    def fwd(prec=0, B=4, H=2, N=16, D=64, q=p, table=p, tdt=0, index=p, u8=None, ids=None, nW=0, strides=st, bias=p, scale=0.125):
        return lib.fa_window_attention_rel_bias(prec, B, H, N, D, q, p, p, p, strides, table, tdt, index, u8, ids, nW,
                                                scale, bias, None, None)

    assert fwd(prec=3) == _lib.FA_ERR_INVALID
    assert fwd(D=32) == _lib.FA_ERR_UNSUPPORTED and b"head_dim" in lib.fa_last_error()
    assert fwd(N=145) == _lib.FA_ERR_UNSUPPORTED and b"144" in lib.fa_last_error()
    assert fwd(N=0) == _lib.FA_ERR_INVALID
    assert fwd(q=None) == _lib.FA_ERR_INVALID and b"null" in lib.fa_last_error()
    assert fwd(q=ctypes.c_void_p((1 << 20) + 2)) == _lib.FA_ERR_INVALID and b"aligned" in lib.fa_last_error()
    assert fwd(table=None) == _lib.FA_ERR_INVALID and fwd(index=None) == _lib.FA_ERR_INVALID
    assert fwd(tdt=2) == _lib.FA_ERR_INVALID and b"table dtype" in lib.fa_last_error()
    assert fwd(u8=p, ids=p, nW=1) == _lib.FA_ERR_INVALID and b"at most one" in lib.fa_last_error()
    assert fwd(ids=p, nW=0) == _lib.FA_ERR_INVALID and b"nW" in lib.fa_last_error()
    assert fwd(B=1 << 30, H=4) == _lib.FA_ERR_INVALID and b"tiles" in lib.fa_last_error()
    bad = (ctypes.c_int64 * 21)(*([60] * 21))
    assert fwd(strides=bad) == _lib.FA_ERR_INVALID and b"16 bytes" in lib.fa_last_error()
    for bad_scale in (0.0, float("nan"), float("inf"), 1e-35):
        assert fwd(scale=bad_scale) == _lib.FA_ERR_INVALID and b"scale" in lib.fa_last_error()
    assert lib.fa_window_attention_rel_bias_state(0, 3, 5) == 3 * 144 * 144 * 4 + 5 * 144
    assert lib.fa_window_attention_rel_bias_state(1, 3, 0) == 2 * 3 * 144 * 144 * 4
    assert lib.fa_window_attention_rel_bias_state(0, 0, 5) == _lib.FA_ERR_INVALID
    assert lib.fa_window_attention_rel_bias_state(2, 1, 0) == _lib.FA_ERR_INVALID
    assert fwd(bias=None) == _lib.FA_ERR_INVALID and b"state buffer" in lib.fa_last_error()
    assert fwd(B=0, q=None) == _lib.FA_OK

    def bwd(stats=p, order=p, nb=5, ws=p, nbytes=1 << 40, tdt=0, bias=p):
        return lib.fa_window_attention_rel_bias_backward(0, 4, 2, 16, 64, p, p, p, p, p, p, p, st, None, None, 0, 0.125,
                                                         bias, stats, order, p, nb, p, tdt, ws, nbytes, None)

    assert bwd(bias=None) == _lib.FA_ERR_INVALID and b"state buffer" in lib.fa_last_error()
    assert bwd(tdt=2) == _lib.FA_ERR_INVALID and b"table dtype" in lib.fa_last_error()
    assert bwd(stats=None) == _lib.FA_ERR_INVALID and b"statistics" in lib.fa_last_error()
    assert bwd(order=None) == _lib.FA_ERR_INVALID and b"bucket lists" in lib.fa_last_error()
    assert bwd(nb=0) == _lib.FA_ERR_INVALID
    assert bwd(ws=None) == _lib.FA_ERR_INVALID and b"workspace" in lib.fa_last_error()
    assert bwd(nbytes=16) == _lib.FA_ERR_INVALID and b"workspace" in lib.fa_last_error()
    assert lib.fa_window_attention_rel_bias_workspace(4, 2, 145) == _lib.FA_ERR_INVALID
    assert lib.fa_window_attention_rel_bias_workspace(4, 2, 16) >= (4 * 2 + 1) * 16 * 16 * 4


def test_clamped_window_reads_the_full_windows_buckets():
    full, small = fa.RelativeBuckets.window((2, 6, 12)), fa.RelativeBuckets.window((2, 3, 4), table_window=(2, 6, 12))
    assert small.num_buckets == full.num_buckets and small.tokens == 24
    # tokens of the small window sit at the same offsets inside the full one
    pos = [(c * 6 + h) * 12 + w for c in range(2) for h in range(3) for w in range(4)]
    assert torch.equal(small.index, full.index[pos][:, pos])
    with pytest.raises(ValueError, match="smaller than the window"):
        fa.RelativeBuckets.window((2, 6, 12), table_window=(2, 6, 11))

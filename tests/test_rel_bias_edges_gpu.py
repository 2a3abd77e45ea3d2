"""Edges of window attention with a relative position bias on the GPU: the calls that its documentation
allows and that the parity tests leave out."""

from __future__ import annotations

import pytest
import torch

import flash_aurora_b200 as fa
from test_rel_bias_gpu import _inputs

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("train", [False, True])
def test_buckets_dropped_while_another_stream_reads_them(train):
    """Buckets built on one stream, used on a second whose work is held back, and dropped: the first stream's
    next allocations must not get their memory. Nothing is written into those allocations."""
    q, k, v, dout, table, index = _inputs(3, 2, 100, BF16, seed=1)
    q = q.requires_grad_(train)
    table = table.requires_grad_(train)
    builder, user = torch.cuda.Stream(), torch.cuda.Stream()

    def call(buckets):
        out = fa.window_attn_rel_bias(q, k, v, table, buckets)
        return torch.autograd.grad(out, (q, table), dout) if train else out

    def ranges(tensors):
        return [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in tensors]

    torch.cuda.synchronize()
    with torch.cuda.stream(user):
        call(fa.RelativeBuckets(index, table.shape[0]))  # what is loaded or allocated once
    torch.cuda.synchronize()
    with torch.cuda.stream(builder):
        buckets = fa.RelativeBuckets(index, table.shape[0])
    read = [buckets.index] + ([buckets.order, buckets.offsets] if train else [])
    mine = ranges(read)
    sizes = [t.numel() for t in read]
    del read
    with torch.cuda.stream(user):
        torch.cuda._sleep(400_000_000)  # about a fifth of a second
        result = call(buckets)
    del buckets
    with torch.cuda.stream(builder):
        fresh = [torch.empty(n, dtype=torch.int32, device="cuda") for n in sizes for _ in range(8)]
    assert not user.query()  # the calls are still behind the wait
    for lo, hi in ranges(fresh):
        assert all(hi <= a or b <= lo for a, b in mine)
    torch.cuda.synchronize()
    want = call(fa.RelativeBuckets(index, table.shape[0]))
    for a, b in zip(result if train else [result], want if train else [want]):
        assert torch.equal(a, b)


def test_transforms_are_refused():
    from torch.autograd import forward_ad
    from torch.func import grad, jvp, vmap
    q, k, v, _, table, index = _inputs(2, 2, 20, FP32, seed=2)
    b = fa.RelativeBuckets(index, table.shape[0])
    x, p = torch.randn(2, 5, 64, device="cuda"), torch.randn(64, device="cuda")
    for f, a in ((lambda t: fa.window_attn_rel_bias(t, k, v, table, b), q),
                 (lambda t: fa.window_attn_rel_bias(q, k, v, t, b), table),
                 (lambda t: fa.block_prenorm(t, p), x), (lambda t: fa.block_prenorm(x, t), p)):
        with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            f(forward_ad.make_dual(a, torch.ones_like(a)))
        with pytest.raises((RuntimeError, NotImplementedError)):
            jvp(f, (a,), (a,))
        with pytest.raises(RuntimeError):
            grad(lambda t: f(t).sum())(a)
        with pytest.raises((RuntimeError, ValueError)):
            vmap(f)(torch.stack((a, a)))
        assert torch.isfinite(f(a)).all()


def test_block_path_makes_no_graph(monkeypatch):
    """The block's path is inference: in grad mode too, the attention gets nothing that requires grad, and the
    output has the bits that it has without grad mode."""
    from flash_aurora_b200 import swin3d
    blk = swin3d.Swin3DTransformerBlock(dim=64, num_heads=1, time_dim=32, window_size=(2, 3, 4), shift_size=(1, 1, 2),
                                        precision="fp32", rel_pos_bias=True)
    swin3d.init_random_weights_(blk)
    with torch.no_grad():
        blk.attn.relative_position_bias_table.normal_()
    blk = blk.cuda()
    g = torch.Generator(device="cuda").manual_seed(3)
    x, c = torch.randn(1, 4 * 6 * 8, 64, device="cuda", generator=g), torch.randn(1, 32, device="cuda", generator=g)
    with torch.no_grad():
        want = blk(x, c, (4, 6, 8))
    seen = []
    call = swin3d.window_attn_rel_bias_qkvpacked

    def attention(*args, **kw):
        seen.append(call(*args, **kw))
        return seen[-1]

    monkeypatch.setattr(swin3d, "window_attn_rel_bias_qkvpacked", attention)
    assert torch.is_grad_enabled() and blk.attn.qkv.weight.requires_grad
    got = blk(x, c, (4, 6, 8))
    assert len(seen) == 1 and not seen[0].requires_grad
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_infinity_in_v_and_dout_reaches_its_own_column_only(dtype, value):
    """out[:, d] and dv[:, d] sum over column d of v and of dout alone, so every other column has the bits that it
    has with a zero in that place. The other (window, head) pairs keep all of theirs."""
    N = 40
    q, k, v, dout, table, index = _inputs(3, 2, N, dtype, seed=4)
    ids = torch.zeros(1, N, dtype=torch.uint8, device="cuda")
    ids[0, 30:] = 1
    spots = {(0, 1): (3, 5), (2, 0): (N - 1, 63), (1, 1): (35, 0)}  # (window, head): (token, column)

    def run(x):
        vv, gg = v.clone(), dout.clone()
        for (w, h), (i, d) in spots.items():
            vv[w, h, i, d] = x
            gg[w, h, i, d] = x
        leaves = [t.clone().requires_grad_(True) for t in (q, k, vv)]
        out = fa.window_attn_rel_bias(*leaves, table, fa.RelativeBuckets(index, table.shape[0]), group_ids=ids)
        return (out.detach(), *torch.autograd.grad(out, leaves, gg))

    clean, got = run(0.0), run(value)
    for name, a, b in (("out", got[0], clean[0]), ("dv", got[3], clean[3])):
        keep = torch.ones_like(a, dtype=torch.bool)
        for (w, h), (i, d) in spots.items():
            keep[w, h, :, d] = False
            assert not torch.isfinite(a[w, h, i, d]), (name, w, h)  # its own token at least
        assert torch.equal(a[keep], b[keep]), (name, float((a[keep] - b[keep]).abs().max()))
    for a, b in zip(got, clean):
        assert torch.equal(a[0, 0], b[0, 0]) and torch.equal(a[1, 0], b[1, 0]) and torch.equal(a[2, 1], b[2, 1])

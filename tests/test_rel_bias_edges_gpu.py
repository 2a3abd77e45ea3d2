"""Edges of window attention with a relative position bias on the GPU: the calls that its documentation
allows and that the parity tests leave out.

Where a test compares with the float64 definition without a bound of its own, the bounds are those that
test_rel_bias_gpu.py derives: 1.42 * 2^-8 of an output's norm in bf16, 1e-5 in fp32 and for the table's
gradient (of its norm, or of 1).
"""

from __future__ import annotations

import math

import pytest
import torch

import flash_aurora_b200 as fa
from _rel_bias_ref import reference
from test_rel_bias_gpu import TOL, _check, _inputs, _run, rel_l2

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


def _region_ids(counts, N, g):
    """Windows of these numbers of regions (N at most), with arbitrary ids in arbitrary places."""
    rows = []
    for c in counts:
        names = torch.randperm(256, device="cuda", generator=g)[:min(c, N)]
        at = torch.arange(N, device="cuda")[torch.randperm(N, device="cuda", generator=g)] % names.numel()
        rows.append(names[at])
    return torch.stack(rows).to(torch.uint8)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("N", [129, 144])
@pytest.mark.parametrize("kind", ["none", "ids", "bytes"])
def test_masks_over_many_tiles_of_a_block(kind, N, dtype):
    """960 tiles, 6 or 7 in a row for each persistent block, so that every ring and phase of the kernels wraps. The
    windows' numbers of regions change from tile to tile, and with them the bf16 kernels' mask products: from none to
    more than there is room for at once.

    The bounds hold: a window whose tokens see only themselves has dS = 0, where fp32 leaves P (dP - delta) with
    up to 2e-6 of dP's 8 deviations. That is a fifth of the windows; the others' rows of dS have norms of 8 / sqrt(keys
    that count), 2 at least, so the share of the norm is below 1.6e-5 * sqrt(1 / 5) / 2 = 4e-6."""
    Bwin, H = 60, 16
    q, k, v, dout, table, index = _inputs(Bwin, H, N, dtype, seed=N)
    g = torch.Generator(device="cuda").manual_seed(6)
    kw, ids, mask = {}, None, None
    if kind == "ids":
        ids = _region_ids([1, 2, 17, 65, 144, 1, 144, 2, 65, 1, 17, 16, 144], N, g)
        kw["group_ids"] = ids
    elif kind == "bytes":
        mask = torch.rand(7, N, N, device="cuda", generator=g) < 0.3
        mask[2] = False
        kw["bias"] = torch.where(mask, -100.0, 0.0)
    got = _run(q, k, v, table, index, dout, **kw)
    _check(got, reference(q, k, v, table, index, 0.125, dout, ids, mask), dtype)
    assert fa.device_status()["attention"] == 0


def test_one_token_fp32():
    """One key: out = v, dv = dout, and dS = P (dP - delta) = 0, of which fp32 may leave the difference of two
    sums of the same 64 products, 2^-21 of their magnitudes each (a split loses up to 2^-23 per operand, the dropped
    product 2^-22, the sum's roundings as much again)."""
    q, k, v, dout, table, index = _inputs(5, 3, 1, FP32, seed=7)
    out, dq, dk, dv, dtable = _run(q, k, v, table, index, dout)
    assert rel_l2(out, v) <= 2.0 ** -21
    assert rel_l2(dv, dout) <= TOL[FP32]  # P is recomputed, from logits of a few units
    dS = 2.0 ** -20 * (dout.double() * v.double()).abs().sum(-1, keepdim=True)
    assert bool((dq.double().abs() <= 0.125 * dS * k.double().abs()).all())
    assert bool((dk.double().abs() <= 0.125 * dS * q.double().abs()).all())
    assert bool((dtable.double().abs() <= dS.sum((0, 2, 3))).all())


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("scale", [0.05, 0.2, -0.1])
@pytest.mark.parametrize("kind", ["ids", "bytes"])
def test_scales(scale, kind, dtype):
    """Scales other than 1 / 8, at which a masked logit still gets -100. A logit's error, 2^-21 of its terms' sum (41)
    times the scale, stays below 4e-6, inside the bound's 1e-5."""
    N = 70
    q, k, v, dout, table, index = _inputs(6, 3, N, dtype, seed=8)
    g = torch.Generator(device="cuda").manual_seed(1)
    ids = mask = None
    if kind == "ids":
        ids = _region_ids([3, 20, 1], N, g)
    else:
        mask = torch.rand(2, N, N, device="cuda", generator=g) < 0.5
    kw = {"group_ids": ids} if mask is None else {"bias": torch.where(mask, -100.0, 0.0)}
    got = _run(q, k, v, table, index, dout, scale_qk=scale, **kw)
    _check(got, reference(q, k, v, table, index, scale, dout, ids, mask), dtype)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("scale", [0.125, 0.39, -0.195, 3.0, 1e-4])
@pytest.mark.parametrize("kind", ["ids", "bytes"])
def test_masked_logits_get_minus_100_at_any_scale(kind, scale, dtype):
    """Two keys, the other one masked and its bias 95 or 98 above: its weight w = 1 / (1 + e^5) or 1 / (1 + e^2) shows
    the -100. The bf16 kernels' region masks add a sum of two bf16 numbers, good to 2^-17 of 100, so to 7.7e-4 of w;
    P and the output are rounded, 2^-8 each. fp32: three roundings of numbers between 128 and 256, half of 2^-16 each,
    times ln 2: 1.6e-5 of w, and 1e-6 for the sums."""
    q = torch.zeros(1, 1, 2, 64, device="cuda", dtype=dtype)
    v = torch.zeros_like(q)
    v[0, 0, 0, 0] = v[0, 0, 1, 1] = 1.0
    b = fa.RelativeBuckets(torch.arange(4, device="cuda").view(2, 2), 4)
    if kind == "ids":
        kw = {"group_ids": torch.tensor([[3, 9]], dtype=torch.uint8, device="cuda")}
    else:
        kw = {"bias": torch.tensor([[[0.0, -100.0], [-100.0, 0.0]]], device="cuda")}
    tol = 2 * 2.0 ** -8 + 7.7e-4 if dtype == BF16 else 1.7e-5
    for lift in (95.0, 98.0):
        table = torch.tensor([[0.0], [lift], [lift], [0.0]], device="cuda")
        w = 1.0 / (1.0 + math.exp(100.0 - lift))
        out = fa.window_attn_rel_bias(q, q, v, table, b, scale_qk=scale, **kw)[0, 0].double()
        for got, want in ((out[0, 1], w), (out[1, 0], w), (out[0, 0], 1 - w), (out[1, 1], 1 - w)):
            assert abs(float(got) - want) <= tol * want, (lift, float(got), want)


def test_nan_and_infinity_in_bf16_queries():
    """A query's row only, also where the second accumulator block reads rows 88 to 127 again and past the tile."""
    N = 144
    q, k, v, _, table, index = _inputs(2, 2, N, BF16, seed=9)
    b = fa.RelativeBuckets(index, table.shape[0])
    ids = (torch.arange(N, device="cuda") // 50).to(torch.uint8).view(1, N)
    for kw in ({}, {"group_ids": ids}, {"bias": torch.where(ids[:, :, None] != ids[:, None, :], -100.0, 0.0)}):
        clean = fa.window_attn_rel_bias(q, k, v, table, b, **kw)
        q2 = q.clone()
        bad = torch.zeros(2, 2, N, dtype=torch.bool, device="cuda")
        for w, h, i, x in ((0, 1, 3, "nan"), (1, 0, 100, "nan"), (1, 0, 143, "inf"), (0, 0, 130, "nan"), (1, 1, 127, "inf")):
            q2[w, h, i, 7 * w + h] = float(x)
            bad[w, h, i] = True
        out = fa.window_attn_rel_bias(q2, k, v, table, b, **kw)
        assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], clean[~bad])


def test_bf16_output_is_that_of_p_rounded_once():
    """The bf16 kernel's one rounding besides the output's is P's, before P V. With it made in float64 too, what is
    left are values that fp32 puts on the other side of a border: one P in a thousand (errors of 2e-6 against steps
    of 2^-8), sqrt(1e-3) 2^-8 = 1.2e-4 of the output, and outputs near a border of their own, sqrt(1.2e-4 * 2^-8) =
    7e-4. The distance to the definition itself is 2.1e-3, to that of the output's rounding alone 1.7e-3."""
    q, k, v, _, table, index = _inputs(20, 4, 144, BF16, seed=10)
    out = fa.window_attn_rel_bias(q, k, v, table, fa.RelativeBuckets(index, table.shape[0]))
    x = q.double() @ k.double().transpose(-1, -2) * 0.125 + table.double()[index].permute(2, 0, 1)
    e = torch.exp(x - x.amax(-1, keepdim=True))
    want = ((e.to(BF16).double() @ v.double()) / e.sum(-1, keepdim=True)).to(BF16)
    assert rel_l2(out, want) <= 7e-4


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_overlapping_unaligned_and_repeated(dtype):
    """Windows that overlap in memory, a packed tensor at an odd address, a backward pass run twice."""
    T, H, N = 48, 2, 16
    g = torch.Generator(device="cuda").manual_seed(11)
    base = torch.randn(T, H * 64, device="cuda", generator=g).to(dtype)
    table, index = torch.randn(31, H, device="cuda", generator=g), torch.randint(0, 31, (N, N), device="cuda", generator=g)
    b = fa.RelativeBuckets(index, 31)
    windows = base.unfold(0, N, 4).permute(0, 2, 1).view(-1, N, H, 64).transpose(1, 2)
    assert not windows.is_contiguous()
    out = fa.window_attn_rel_bias(windows, windows, windows, table, b)
    c = windows.contiguous()
    assert torch.equal(out, fa.window_attn_rel_bias(c, c, c, table, b))
    leaf = base.clone().requires_grad_(True)
    w = leaf.unfold(0, N, 4).permute(0, 2, 1).view(-1, N, H, 64).transpose(1, 2)
    dout = torch.randn(out.shape, device="cuda", generator=g).to(dtype)
    o = fa.window_attn_rel_bias(w, w, w, table, b)
    one = torch.autograd.grad(o, w, dout, retain_graph=True)[0]
    ref = reference(c, c, c, table, index, 0.125, dout)
    assert rel_l2(one, ref[1] + ref[2] + ref[3]) <= (2 if dtype == BF16 else 1) * TOL[dtype]  # bf16: two more roundings
    assert torch.equal(one, torch.autograd.grad(o, w, dout)[0])

    qkv = torch.randn(5, N, 3 * H * 64, device="cuda", generator=g).to(dtype)
    odd = torch.zeros(qkv.numel() + 1, device="cuda", dtype=dtype)[1:].view(qkv.shape)
    odd.copy_(qkv)
    assert odd.data_ptr() % 16
    res = []
    for t in (qkv, odd):
        t = t.detach().requires_grad_(True)
        o = fa.window_attn_rel_bias_qkvpacked(t, H, table, b, output_layout="bnc")
        go = torch.ones(o.numel() + 1, device="cuda", dtype=dtype)[1:].view(o.shape)
        res.append((o.detach(), torch.autograd.grad(o, t, go)[0]))
    assert all(torch.equal(a, z) for a, z in zip(*res))


def test_buckets_without_pairs():
    """Far more buckets than pairs: the empty ones have a gradient of zero."""
    q, k, v, dout, table, _ = _inputs(4, 3, 12, FP32, seed=12, nb=70001)
    g = torch.Generator(device="cuda").manual_seed(2)
    index = torch.randint(0, 70001, (12, 12), device="cuda", generator=g)
    index[0, 0], index[11, 11] = 0, 70000
    got = _run(q, k, v, table, index, dout)
    _check(got, reference(q, k, v, table, index, 0.125, dout), FP32)
    empty = torch.ones(70001, dtype=torch.bool, device="cuda")
    empty[index.reshape(-1)] = False
    assert float(got[4][empty].abs().max()) == 0.0


@pytest.mark.parametrize("precision,tol", [("fp32", 1e-6), ("bf16_mixed", 5e-3)])
def test_bands_read_the_bias(precision, tol):
    """A stage with a bias on two and three latitude bands (threads that exchange through the host) against the whole
    field; tolerances as for the stages without a bias."""
    from flash_aurora_b200 import sharding
    from flash_aurora_b200.swin3d import BasicLayer3D
    field_res, ws, dim = (4, 36, 72), (2, 6, 12), 128
    C, H, W = field_res
    torch.manual_seed(5)
    layer = BasicLayer3D(dim=dim, depth=2, num_heads=2, ws=ws, time_dim=dim, precision=precision, rel_pos_bias=True)
    with torch.no_grad():
        for name, p in layer.named_parameters():
            p.normal_(0.0, 1.0 if "bias_table" in name else 0.02)
    layer = layer.cuda().eval()
    g = torch.Generator().manual_seed(9)
    x, c = torch.randn(1, C * H * W, dim, generator=g).cuda(), torch.randn(1, dim, generator=g).cuda()
    with torch.no_grad():
        want = layer(x, c, field_res)[0].view(1, C, H, W, dim)
    x5 = x.view(1, C, H, W, dim)
    for world in (2, 3):
        def fn(rank, ring):
            ctx = sharding.BandContext(field_res, ws, rank, world, ring=ring, timeout_s=60)
            a, b = ctx.h_begin, ctx.h_end
            with torch.no_grad():
                yb, _ = layer(x5[:, :, a:b].reshape(1, -1, dim).contiguous(), c, ctx.res, band=ctx)
            torch.cuda.synchronize()
            return yb.view(1, C, b - a, W, dim)

        got = torch.cat(sharding.run_ranks(world, fn, timeout_s=120), dim=2)
        assert rel_l2(got, want) <= tol

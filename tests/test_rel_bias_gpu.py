"""GPU parity of window attention with a relative position bias, forward and gradients, against the
definition in float64 on the same (rounded) inputs.

Tolerances are on the relative L2 norm of each output.

* bf16 tensors: the output is rounded once (at most half a step, 2^-9 of a value whose leading bit
  is 1, 2^-8 at worst), and P, respectively dS, once more before its product: two roundings of at
  most 2^-8 each in quadrature, 1.42 * 2^-8 = 5.6e-3, if every rounding error were the largest one
  and none cancelled.
* fp32 tensors: operands of 22 bits keep about 2^-21 of a product and the logits reach a few tens, whose
  rounding (2^-24 * 32 = 2e-6 of a logit, so of a probability) dominates: 1e-5.
* the table's gradient of bf16 tensors has no rounding but the fp32 ones: 1e-5 too. A sum that
  cancels to a small part of its terms is measured against the terms: the bound is on the norm over all
  buckets, and holds where the buckets' sums do not all cancel.
"""

from __future__ import annotations

import pytest
import torch

import flash_aurora_b200 as fa
from _rel_bias_ref import reference

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32
TOL = {BF16: 1.42 * 2.0 ** -8, FP32: 1e-5}
TABLE_TOL = 1e-5


def rel_l2(x, ref):
    ref = ref.double()
    return float((x.double() - ref).norm() / ref.norm().clamp(min=1e-30))


def _inputs(Bwin, H, N, dtype, seed=0, nb=None, table_dtype=FP32, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k, v, dout = (torch.randn(Bwin, H, N, 64, device="cuda", generator=g).to(dtype) for _ in range(4))
    nb = nb or 2 * N - 1
    table = (torch.randn(nb, H, device="cuda", generator=g) * std).to(table_dtype)
    index = torch.randint(0, nb, (N, N), device="cuda", generator=g)
    return q, k, v, dout, table, index


def _run(q, k, v, table, index, dout, **kw):
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v, table)]
    out = fa.window_attn_rel_bias(*leaves, fa.RelativeBuckets(index, table.shape[0]), **kw)
    return (out.detach(), *torch.autograd.grad(out, leaves, dout))


def _check(got, ref, dtype, table_tol=TABLE_TOL):
    for name, x, r in zip(("out", "dq", "dk", "dv"), got, ref):
        assert x.dtype == dtype and x.shape == r.shape
        if float(r.norm()) < 1e-6 * r.numel() ** 0.5:  # one key: dq and dk are zero up to rounding
            assert float(x.double().abs().max()) < 1e-3 if dtype == BF16 else 1e-5, name
            continue
        assert rel_l2(x, r) <= TOL[dtype], (name, rel_l2(x, r))
    assert got[4].shape == ref[4].shape
    scale = max(1.0, float(ref[4].norm()))
    assert float((got[4].double() - ref[4]).norm()) <= table_tol * scale, float((got[4].double() - ref[4]).norm()) / scale


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("N", [1, 2, 7, 8, 15, 16, 17, 31, 64, 65, 98, 127, 128, 129, 136, 143, 144])
def test_lengths(N, dtype):
    q, k, v, dout, table, index = _inputs(5, 3, N, dtype, seed=N)
    got = _run(q, k, v, table, index, dout)
    _check(got, reference(q, k, v, table, index, 0.125, dout), dtype)
    assert fa.device_status()["attention"] == 0


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("Bwin,H", [(1, 1), (1, 7), (150, 1), (37, 5), (2, 160), (400, 2)])
def test_tile_counts(Bwin, H, dtype):
    """Fewer tiles than SMs, heads that end inside a block's range, several heads in one block."""
    q, k, v, dout, table, index = _inputs(Bwin, H, 48, dtype, seed=3)
    _check(_run(q, k, v, table, index, dout), reference(q, k, v, table, index, 0.125, dout), dtype)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("N", [24, 33, 144])
@pytest.mark.parametrize("kind", ["ids", "many_ids", "bias", "all"])
def test_masks(N, kind, dtype):
    q, k, v, dout, table, index = _inputs(6, 2, N, dtype, seed=5)
    g = torch.Generator(device="cuda").manual_seed(9)
    kw, ids, mask = {}, None, None
    if kind == "ids":
        ids = torch.randint(0, 4, (3, N), device="cuda", generator=g, dtype=torch.uint8)
        ids[0] = 7  # one region: nothing masked
        kw["group_ids"] = ids
    elif kind == "many_ids":  # every token a region of its own: only the diagonal is unmasked
        ids = torch.arange(N, device="cuda").to(torch.uint8).repeat(2, 1)
        kw["group_ids"] = ids
    elif kind == "bias":
        mask = torch.rand(3, N, N, device="cuda", generator=g) < 0.4
        mask[1, 2] = True  # a row with every key masked: -100 everywhere, so as if unmasked
        kw["bias"] = torch.where(mask, -100.0, 0.0)
    else:
        mask = torch.ones(1, N, N, device="cuda", dtype=torch.bool)
        kw["bias"] = torch.full((1, N, N), torch.finfo(torch.float32).min, device="cuda")
    _check(_run(q, k, v, table, index, dout, **kw), reference(q, k, v, table, index, 0.125, dout, ids, mask), dtype)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_packed_equals_split_and_both_layouts(dtype):
    Bwin, H, N = 9, 4, 98
    q, k, v, dout, table, index = _inputs(Bwin, H, N, dtype, seed=11)
    b = fa.RelativeBuckets(index, table.shape[0])
    ref = _run(q, k, v, table, index, dout, scale_qk=0.2)
    qkv0 = torch.stack((q, k, v)).permute(1, 3, 0, 2, 4).reshape(Bwin, N, 3 * H * 64).contiguous()
    for layout in ("bhnd", "bnc"):
        qkv, t = qkv0.clone().requires_grad_(True), table.clone().requires_grad_(True)
        out = fa.window_attn_rel_bias_qkvpacked(qkv, H, t, b, scale_qk=0.2, output_layout=layout)
        go = dout if layout == "bhnd" else dout.transpose(1, 2).reshape(Bwin, N, H * 64)
        dqkv, dt = torch.autograd.grad(out, (qkv, t), go)
        o = out if layout == "bhnd" else out.view(Bwin, N, H, 64).transpose(1, 2)
        assert torch.equal(o, ref[0])
        assert torch.equal(dqkv.view(Bwin, N, 3, H, 64).permute(2, 0, 3, 1, 4), torch.stack(ref[1:4]))
        assert torch.equal(dt, ref[4])
        with torch.no_grad():
            assert torch.equal(fa.window_attn_rel_bias_qkvpacked(qkv0, H, table, b, scale_qk=0.2, output_layout=layout),
                               out)


def test_strided_broadcast_and_unaligned_inputs():
    Bwin, H, N = 4, 3, 40
    q, k, v, dout, table, index = _inputs(Bwin, H, N, BF16, seed=12)
    want = _run(q, k, v, table, index, dout)
    wide = torch.zeros(Bwin, N, H, 72, device="cuda", dtype=BF16)
    wide[..., :64] = q.transpose(1, 2)
    odd = torch.zeros(q.numel() + 1, device="cuda", dtype=BF16)[1:].view(q.shape)
    odd.copy_(k)
    qs, vs = wide[..., :64].transpose(1, 2), v.transpose(1, 2).contiguous().transpose(1, 2)
    leaves = [t.detach().requires_grad_(True) for t in (qs, odd, vs, table)]
    out = fa.window_attn_rel_bias(*leaves, fa.RelativeBuckets(index, table.shape[0]))
    got = torch.autograd.grad(out, leaves, dout.transpose(1, 2).contiguous().transpose(1, 2))
    for a, b in zip((out, *got), want):
        assert torch.equal(a, b)
    # one value tensor shared by all heads, and a gradient broadcast from a scalar sum
    v1 = v[:, :1].clone().requires_grad_(True)
    leaves = [q, k, v1.expand(Bwin, H, N, 64), table]
    out = fa.window_attn_rel_bias(*leaves, fa.RelativeBuckets(index, table.shape[0]))
    (dv1,) = torch.autograd.grad(out.sum(), v1)
    ref = reference(q, k, v1.expand(Bwin, H, N, 64), table, index, 0.125, torch.ones_like(dout))
    assert rel_l2(dv1, ref[3].sum(1, keepdim=True)) <= TOL[BF16]


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_large_and_lowest_bias_values(dtype):
    Bwin, H, N = 3, 2, 50
    q, k, v, dout, table, index = _inputs(Bwin, H, N, dtype, seed=13, nb=40)
    table[3], table[4] = float("-inf"), torch.finfo(torch.float32).min
    table[5] = 30.0
    index[7, :] = 4  # a row of the lowest value only: the softmax of its scores at that level is uniform
    index[9, 0], index[9, 1:] = 0, 3  # a row with one key left
    got = _run(q, k, v, table, index, dout)
    # In 64 bits the lowest value of fp32 swamps the scores as it does in 32.
    ref = list(reference(q, k, v, table, index, 0.125, dout))
    rows = [i for i in range(N) if i != 7]
    assert rel_l2(got[0][:, :, rows], ref[0][:, :, rows]) <= TOL[dtype]
    assert rel_l2(got[0][:, :, 7], v.double().mean(2)) <= TOL[dtype]
    assert all(bool(torch.isfinite(x).all()) for x in got)


def test_bf16_table_and_window_buckets():
    b = fa.RelativeBuckets.window((2, 6, 12), "cuda")
    assert b.num_buckets == 3 * 11 * 23 and b.tokens == 144
    q, k, v, dout, table, _ = _inputs(10, 4, 144, BF16, seed=14, nb=b.num_buckets, table_dtype=BF16, std=0.5)
    got = _run(q, k, v, table, b.index, dout)
    ref = reference(q, k, v, table, b.index, 0.125, dout)
    _check((*got[:4], got[4].double()), ref, BF16, table_tol=2.0 ** -8)
    assert got[4].dtype == BF16


def test_gradient_matches_differences():
    """d(sum(out * dout)) along random directions, by central differences of the float64 definition at
    the fp32 kernel's inputs. The difference quotient's own error is h^2 times a third derivative plus
    rounding / h, below 1e-6 of the gradient's norm at h = 1e-4; the kernel's is 1e-5 (above)."""
    from _rel_bias_ref import attention64
    q, k, v, dout, table, index = _inputs(2, 2, 30, FP32, seed=15)
    grads = _run(q, k, v, table, index, dout)[1:]
    base = [t.double() for t in (q, k, v, table)]
    g = torch.Generator(device="cuda").manual_seed(1)
    for i, gr in enumerate(grads):
        d = torch.randn(gr.shape, device="cuda", generator=g, dtype=torch.float64)
        d = gr.double() / gr.double().norm() + 0.1 * d / d.norm()
        f = []
        for h in (1e-4, -1e-4):
            x = list(base)
            x[i] = x[i] + h * d
            f.append(float((attention64(*x, index, 0.125) * dout.double()).sum()))
        slope = (f[0] - f[1]) / 2e-4
        assert abs(slope - float((gr.double() * d).sum())) <= 1.2e-5 * float(gr.double().norm()), i


def test_empty_batch_and_partial_gradients():
    q, k, v, dout, table, index = _inputs(4, 2, 20, BF16, seed=16)
    b = fa.RelativeBuckets(index, table.shape[0])
    e = q[:0].clone().requires_grad_(True)
    t = table.clone().requires_grad_(True)
    out = fa.window_attn_rel_bias(e, k[:0], v[:0], t, b)
    assert out.shape == (0, 2, 20, 64)
    de, dt = torch.autograd.grad(out, (e, t), out.detach())
    assert de.shape == e.shape and float(dt.abs().max()) == 0.0
    want = _run(q, k, v, table, index, dout)
    for i in range(4):
        leaves = [x.detach().clone().requires_grad_(j == i) for j, x in enumerate((q, k, v, table))]
        out = fa.window_attn_rel_bias(*leaves, b)
        (gi,) = torch.autograd.grad(out, leaves[i], dout)
        assert torch.equal(gi, want[1 + i])


def test_same_bits_and_side_stream():
    q, k, v, dout, table, index = _inputs(120, 3, 144, BF16, seed=17)
    a = _run(q, k, v, table, index, dout)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = _run(q, k, v, table, index, dout)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_mask_changed_before_backward_is_refused():
    q, k, v, dout, table, index = _inputs(2, 2, 16, BF16, seed=18)
    ids = torch.zeros(2, 16, dtype=torch.uint8, device="cuda")
    q = q.requires_grad_(True)
    out = fa.window_attn_rel_bias(q, k, v, table, fa.RelativeBuckets(index, table.shape[0]), group_ids=ids)
    ids.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, q, dout)


def test_captured_forward_and_backward():
    q, k, v, dout, table, index = _inputs(6, 2, 144, BF16, seed=19)
    b = fa.RelativeBuckets(index, table.shape[0])
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, table)]

    def step():
        out = fa.window_attn_rel_bias(*leaves, b)
        return (out.detach(), *torch.autograd.grad(out, leaves, dout))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for _ in range(2):  # two graphs, each with workspaces of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    with torch.no_grad():
        leaves[0].copy_(q * 0.5)
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    want = _run(q * 0.5, k, v, table, index, dout)
    for o in outs:
        assert all(torch.equal(x, y) for x, y in zip(o, want))


def _uneven(shape, g, bits):
    """Normal values times a power of two per row, 2^-bits to 2^bits."""
    x = torch.randn(*shape, device="cuda", generator=g)
    return x * torch.exp2(torch.randint(-bits, bits + 1, (*shape[:-1], 1), device="cuda", generator=g).float())


@pytest.mark.parametrize("N", [5, 33, 144])
@pytest.mark.parametrize("bits", [20, 40])
def test_rows_of_any_size_fp32(N, bits):
    """Rows of v and dout from 2^-bits to 2^bits, one of zeros, one of denormals, and the largest that dP
    allows (64 terms, 4 deviations of dout's 2^bits, below 2^127) in rows that the mask takes from the others: every element against the sum of the magnitudes of its own terms.

    A logit is off by at most 2^-21 of its terms' magnitudes (a split loses up to 2^-23 per operand, the dropped
    lo lo 2^-22, the sums' roundings as much again), which q and k of deviation 0.5 keep below 4 in sum
    after the scale: 2e-6 of a probability, twice that with the row's sum; a product over tokens adds 2^-21 and
    the roundings of its nine partial sums, 1e-6: 6e-6 for the output and dV. dS takes three such factors (P, dP
    and delta) and the product one more: 2e-5 for dQ and dK. A masked probability (e^-100 and less) is an fp32
    number below 2^-126 with a resolution of 2^-149, half of which is 6e-6 of 2^-133: the terms count it with
    2^-132 more."""
    g = torch.Generator(device="cuda").manual_seed(N + bits)
    B, H = 3, 2
    q, k = (0.5 * torch.randn(B, H, N, 64, device="cuda", generator=g) for _ in range(2))
    v, dout = _uneven((B, H, N, 64), g, bits), _uneven((B, H, N, 64), g, bits)
    v[0, 0, 0] = 0
    dout[1, 0, 1] = 0
    v[1, 1, 2] = 1e-40
    ids = torch.zeros(1, N, dtype=torch.uint8, device="cuda")
    ids[0, N - 1] = 1  # a key for itself only
    v[2, :, N - 1] = 2.0 ** (127 - 6 - 2 - bits)
    dout[2, :, N - 1] = 0
    table = torch.randn(2 * N - 1, H, device="cuda", generator=g)
    index = torch.randint(0, 2 * N - 1, (N, N), device="cuda", generator=g)
    got = _run(q, k, v, table, index, dout, group_ids=ids)
    Q, K, V, G = (t.double() for t in (q, k, v, dout))
    x = Q @ K.transpose(-1, -2) * 0.125 + table.double()[index].permute(2, 0, 1) - 100.0 * (ids[:, :, None] != ids[:, None, :]).double()
    P = torch.softmax(x, -1)
    P_size = P + 2.0 ** -132
    dP = G @ V.transpose(-1, -2)
    size = G.abs() @ V.abs().transpose(-1, -2)  # of dP's terms
    dS = P * (dP - (P * dP).sum(-1, keepdim=True))
    dS_size = P_size * (size + (P_size * size).sum(-1, keepdim=True))
    T = lambda t: t.transpose(-1, -2)  # noqa: E731
    want = {"out": (P @ V, P_size @ V.abs(), 6e-6), "dq": (0.125 * dS @ K, 0.125 * dS_size @ K.abs(), 2e-5),
            "dk": (0.125 * T(dS) @ Q, 0.125 * T(dS_size) @ Q.abs(), 2e-5), "dv": (T(P) @ G, T(P_size) @ G.abs(), 6e-6)}
    for x, (name, (ref, terms, tol)) in zip(got, want.items()):
        assert torch.isfinite(x).all(), name
        worst = ((x.double() - ref).abs() / (terms + 1e-37)).max()
        assert float(worst) <= tol, (name, float(worst))


def test_infinity_and_nan_reach_their_own_rows_only():
    q, k, v, dout, table, index = _inputs(2, 2, 40, FP32)
    clean = _run(q, k, v, table, index, dout)[0]
    q2 = q.clone()
    q2[0, 1, 3, 5], q2[1, 0, 7, 0] = float("nan"), float("inf")
    out = _run(q2, k, v, table, index, dout)[0]
    bad = torch.zeros(2, 2, 40, dtype=torch.bool, device="cuda")
    bad[0, 1, 3] = bad[1, 0, 7] = True
    assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], clean[~bad])

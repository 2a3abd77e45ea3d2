"""Edges of the block norms on the GPU: rows that are not whole 16-byte units, in every type, with gradients; more
batch elements than a grid holds.

Bounds as test_block_norm_gpu.py derives them (2^-8 of an output's norm in bf16, 6e-6 in fp32 for rows whose
deviation is about their size). Narrow rows may have a deviation that is a small part of their largest magnitude:
the mean's rounding then counts that much more in the normalised row and in what is computed from it, so the
fp32 bound is multiplied by the largest such ratio of the rows that are normalised.
"""

from __future__ import annotations

import pytest
import torch

import flash_aurora_b200 as fa
import _block_norm_ref as R
from test_block_norm_gpu import BF16, FP32, NAMES, TOL, _both, _call, _make, rel_l2

pytestmark = pytest.mark.gpu


def _ratio(x, norm):
    """The largest of (magnitude / deviation) over rows."""
    x = x.detach().double()
    dev = x - x.mean(-1, keepdim=True) if norm == "layer" else x
    return float((x.abs().amax(-1) / dev.pow(2).mean(-1).sqrt()).max())


def _check(form, t, douts, norm):
    ref = {n: v.double() for n, v in t.items()}
    more = max(1.0, _ratio(t["x"], norm))
    if form == "between":
        more += _ratio(_call(R, "between", ref, norm=norm)[0], norm)
    results = _both(form, t, douts, norm=norm)
    for name, a, b in results:
        assert a.shape == b.shape, name
        err, size = rel_l2(a, b), float(b.detach().norm())
        if name[1:] in NAMES and size > 0:  # a column's sum may cancel: against sqrt(terms), see the other file
            terms = results[0][1].numel() // b.numel()
            err *= size / max(size, (terms * b.numel()) ** 0.5)
        assert err <= (TOL[BF16] + TOL[FP32] * more if a.dtype == BF16 else TOL[FP32] * more), (name, err, more)


TYPES = [(BF16, FP32), (BF16, BF16), (FP32, FP32), (FP32, BF16)]


@pytest.mark.parametrize("form,dt,rdt", [("before", BF16, BF16), ("before", FP32, FP32),
                                         *((f, *p) for f in ("after", "between") for p in TYPES)])
@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("D", [5, 33, 255, 771, 2047, 4095])
@pytest.mark.parametrize("per_batch", ["none", "mixed"])
def test_ragged_rows(form, norm, D, dt, rdt, per_batch):
    t, d = _make(form, 3, 23, D, dt, rdt, per_batch, seed=D)
    _check(form, t, d, norm)


@pytest.mark.parametrize("dt,out", [(BF16, FP32), (FP32, BF16)])
@pytest.mark.parametrize("D", [64, 771])
def test_gradients_through_another_output_type(dt, out, D):
    t, (dz,) = _make("before", 2, 40, D, dt, FP32, "all", seed=5)
    dz = dz.to(out)
    own = {n: v.clone().requires_grad_(True) for n, v in t.items()}
    ref = {n: v.double().requires_grad_(True) for n, v in t.items()}
    z = fa.block_prenorm(own["x"], own["pre_scale"], own["pre_shift"], out_dtype=out)
    r = R.prenorm(ref["x"], ref["pre_scale"], ref["pre_shift"])
    got = (z, *torch.autograd.grad(z, list(own.values()), dz))
    want = (r, *torch.autograd.grad(r, list(ref.values()), dz.double()))
    assert z.dtype == out
    for i, (a, b) in enumerate(zip(got, want)):
        assert rel_l2(a, b) <= (TOL[BF16] if a.dtype == BF16 else 0.0) + TOL[FP32] * _ratio(t["x"], "layer"), i


@pytest.mark.parametrize("form", ["before", "after", "between"])
@pytest.mark.parametrize("dt,rdt", [(FP32, FP32), (BF16, BF16)])
def test_widest_rows(form, dt, rdt):
    t, d = _make(form, 2, 300, 4096, dt, rdt, "all", seed=1)
    _check(form, t, d, "layer")


@pytest.mark.parametrize("D", [64, 772])
def test_rows_at_odd_addresses(D):
    """Whole units by width but not by address: rows go element by element, gradients included. Forward sums are
    grouped by the same threads but over other columns, so the values differ from the aligned call's by roundings."""
    t, d = _make("between", 2, 40, D, BF16, FP32, "all", seed=2)
    u = dict(t)
    for n in ("x", "residual", "gate"):
        flat = torch.zeros(t[n].numel() + 1, device="cuda", dtype=t[n].dtype)[1:].view(t[n].shape)
        flat.copy_(t[n])
        assert flat.data_ptr() % 16 != 0
        u[n] = flat
    own = {n: v.detach().requires_grad_(True) for n, v in u.items()}
    out = _call(fa, "between", own)
    odd = [torch.zeros(g.numel() + 1, device="cuda", dtype=g.dtype)[1:].view(g.shape).copy_(g) for g in d]
    got = (*out, *torch.autograd.grad(out, list(own.values()), odd))
    want = [b for _, _, b in _both("between", t, d)]
    more = _ratio(t["x"], "layer") + _ratio(want[0], "layer")
    for i, (a, b) in enumerate(zip(got, want)):
        assert rel_l2(a, b) <= (TOL[BF16] if a.dtype == BF16 else 0.0) + TOL[FP32] * more, i


@pytest.mark.parametrize("form", ["before", "after", "between"])
def test_more_batch_elements_than_a_grid_holds(form):
    """70000 batch elements of one row with parameters of their own: the bits of the same call in two halves."""
    B, D = 70000, 16
    t, d = _make(form, B, 1, D, BF16, FP32, "all", seed=3)

    def run(lo, hi):
        own = {n: v[lo:hi].detach().clone().requires_grad_(True) for n, v in t.items()}
        out = _call(fa, form, own)
        return (*(o.detach() for o in out), *torch.autograd.grad(out, list(own.values()), [g[lo:hi] for g in d]))

    whole, first, second = run(0, B), run(0, B // 2), run(B // 2, B)
    for a, b, c in zip(whole, first, second):
        assert torch.equal(a, torch.cat((b, c)))


def test_one_tensor_in_both_places():
    """A block whose output is its own residual: both gradients reach the same leaf."""
    t, d = _make("between", 2, 30, 96, FP32, FP32, "none", seed=4)
    names = [n for n in t if n != "residual"]
    own = {n: t[n].clone().requires_grad_(True) for n in names}
    ref = {n: t[n].double().requires_grad_(True) for n in names}
    o = _call(fa, "between", {**own, "residual": own["x"]})
    r = _call(R, "between", {**ref, "residual": ref["x"]})
    go = torch.autograd.grad(o, list(own.values()), d, retain_graph=True)
    again = torch.autograd.grad(o, list(own.values()), d)
    gr = torch.autograd.grad(r, list(ref.values()), [g.double() for g in d])
    more = _ratio(t["x"], "layer") + _ratio(r[0], "layer")
    for n, a, a2, b in zip(names, go, again, gr):
        assert torch.equal(a, a2) and rel_l2(a, b) <= TOL[FP32] * more, n

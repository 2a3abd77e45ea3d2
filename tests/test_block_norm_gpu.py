"""GPU parity of the norms before / after / between blocks, forward and gradients, against the
definitions in float64 on the same inputs.

Tolerances are on the relative L2 norm of each output. A bf16 output is rounded once: at most half a
step of each value, 2^-8, so 2^-8 of the norm; fp32 arithmetic adds little to that. An fp32 output
follows a chain of about twenty fp32 operations, two reductions among them, of up to 4096 terms each
(errors of a sum in a tree of 8-term chains: about 20 * 2^-24); with the cancellation in (v - mean) of
inputs whose mean is below their deviation, 100 * 2^-24 = 6e-6 bounds it. Column sums add chains of up to
a few hundred rows, whose rounding errors grow like the square root: the same bound. A column sum of n
terms may cancel, as the one column at D = 1 does (38 terms of order one that add up to 5e-4): n terms
of order one, each off by at most 16 roundings of 2^-24, leave an error of up to n 16 2^-24 whatever they
add up to, which for n = 38 is 6e-6 sqrt(n). So a parameter's gradient is measured against its norm or
sqrt(n) a column, whichever is more.
"""

from __future__ import annotations

import pytest
import torch

import flash_aurora_b200 as fa
import _block_norm_ref as R

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32
TOL = {BF16: 2.0 ** -8, FP32: 6e-6}
NAMES = ("scale", "shift", "gate", "residual_scale", "pre_scale", "pre_shift")


def rel_l2(x, ref):
    x, ref = x.detach(), ref.detach().double()
    return float((x.double() - ref).norm() / ref.norm().clamp(min=1e-30))


def _make(form, B, L, D, dt, rdt, per_batch, seed=0, names=NAMES, pdt=FP32):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*s, std=1.0, mean=0.0, dtype=FP32):
        return (torch.randn(*s, device="cuda", generator=g) * std + mean).to(dtype)

    shapes = {"none": (D,), "all": (B, 1, D), "flat": (B, D)}
    t = {"x": rand(B, L, D, mean=0.3, dtype=dt)}
    if form != "before":
        t["residual"] = rand(B, L, D, std=2.0, dtype=rdt)
    use = NAMES[4:] if form == "before" else NAMES[:4] if form == "after" else NAMES
    for i, n in enumerate(use):
        if n in names:
            shape = shapes[per_batch] if per_batch != "mixed" else shapes[("none", "all")[i % 2]]
            t[n] = rand(*shape, std=0.5, mean=0.7 if n in ("gate", "residual_scale") else 0.0, dtype=pdt)
    douts = []
    if form != "before":
        douts.append(rand(B, L, D, dtype=rdt))
    if form != "after":
        douts.append(rand(B, L, D, dtype=dt))
    return t, douts


def _call(mod, form, t, **kw):
    t = dict(t)
    if form == "before":
        f = fa.block_prenorm if mod is fa else R.prenorm
        return (f(t["x"], t.get("pre_scale"), t.get("pre_shift"), **kw),)
    post = {k: t.get(k) for k in ("scale", "shift", "gate")}
    if "residual_scale" in t:
        kw["residual_scale"] = t["residual_scale"]
    if form == "after":
        f = fa.block_postnorm_residual if mod is fa else R.postnorm
        return (f(t["residual"], t["x"], **post, **kw),)
    if mod is fa:
        return fa.block_postnorm_residual_prenorm(t["residual"], t["x"], **post, pre_scale=t.get("pre_scale"),
                                                  pre_shift=t.get("pre_shift"), **kw)
    psb = kw.pop("pre_scale_bias", 1.0)
    y = R.postnorm(t["residual"], t["x"], **post, **kw)
    return y, R.prenorm(y, t.get("pre_scale"), t.get("pre_shift"), scale_bias=psb, eps=kw.get("eps", 1e-5),
                        norm=kw.get("norm", "layer"))


def _both(form, t, douts, **kw):
    """[(name, kernel's, reference)] of every output and gradient."""
    own = {k: v.detach().clone().requires_grad_(True) for k, v in t.items()}
    ref = {k: v.detach().double().requires_grad_(True) for k, v in t.items()}
    o, r = _call(fa, form, own, **kw), _call(R, form, ref, **kw)
    go = torch.autograd.grad(o, list(own.values()), douts)
    gr = torch.autograd.grad(r, list(ref.values()), [d.double() for d in douts])
    with torch.no_grad():
        for a, b in zip(_call(fa, form, own, **kw), o):
            assert torch.equal(a, b)  # the same bits without gradients
    return [(f"out{i}", a, b) for i, (a, b) in enumerate(zip(o, r))] + [
        (f"d{n}", a, b) for n, a, b in zip(t, go, gr)]


def _check(results, like):
    for name, a, b in results:
        assert a.shape == b.shape, name
        err, size = rel_l2(a, b), float(b.detach().norm())
        if name[1:] in NAMES and size > 0:
            n = results[0][1].numel() // b.numel()
            err *= size / max(size, (n * b.numel()) ** 0.5)
        assert err <= TOL[a.dtype], (name, err, like)


@pytest.mark.parametrize("form", ["before", "after", "between"])
@pytest.mark.parametrize("D", [8, 16, 24, 120, 256, 264, 512, 520, 1000, 1024, 2048, 2056, 4096])
def test_widths(form, D):
    t, d = _make(form, 2, 37, D, BF16, FP32, "all", seed=D)
    _check(_both(form, t, d), D)


@pytest.mark.parametrize("form", ["before", "after", "between"])
@pytest.mark.parametrize("D", [1, 3, 7, 31, 33, 100, 255, 513, 771, 1025, 2047, 4095])
def test_odd_widths(form, D):
    t, d = _make(form, 2, 19, D, FP32, FP32, "none", seed=D)
    res = _both(form, t, d, norm="rms")
    if D == 1:  # one channel: the RMS norm's gradient is eps-sized, beside fp32 rounding
        res = [r for r in res if r[0] not in ("dx", "dresidual", "dresidual_scale")]
    _check(res, D)


@pytest.mark.parametrize("form", ["before", "after", "between"])
@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("dt,rdt", [(BF16, FP32), (BF16, BF16), (FP32, FP32), (FP32, BF16)])
@pytest.mark.parametrize("per_batch", ["none", "all", "flat", "mixed"])
def test_types_and_parameter_shapes(form, norm, dt, rdt, per_batch):
    t, d = _make(form, 3, 50, 328, dt, rdt, per_batch, seed=1)
    _check(_both(form, t, d, norm=norm, eps=1e-3), (form, norm))


@pytest.mark.parametrize("form", ["before", "after", "between"])
@pytest.mark.parametrize("B,L", [(1, 1), (1, 2), (7, 1), (1, 5000), (3, 1777), (400, 3)])
def test_row_counts(form, B, L):
    t, d = _make(form, B, L, 96, BF16, FP32, "mixed", seed=2)
    _check(_both(form, t, d), (B, L))


@pytest.mark.parametrize("names", [(), ("gate",), ("scale", "pre_shift"), ("shift", "residual_scale", "pre_scale")])
def test_absent_parameters_and_float_residual_scale(names):
    for form in ("before", "after", "between"):
        t, d = _make(form, 2, 9, 64, FP32, FP32, "none", seed=3, names=names)
        kw = {} if form == "before" else {"scale_bias": 0.25}
        if form != "before" and "residual_scale" not in names:
            kw["residual_scale"] = 0.5
        if form == "between":
            kw["pre_scale_bias"] = 1.5
        _check(_both(form, t, d, **kw), (form, names))


def test_bf16_parameters():
    t, d = _make("between", 2, 33, 128, BF16, BF16, "mixed", seed=4, pdt=BF16)
    _check(_both("between", t, d), "bf16 parameters")


def test_one_of_two_gradients():
    t, d = _make("between", 2, 21, 200, FP32, FP32, "none", seed=5)
    for keep in (0, 1):
        own = {k: v.clone().requires_grad_(True) for k, v in t.items()}
        ref = {k: v.double().requires_grad_(True) for k, v in t.items()}
        go = torch.autograd.grad(_call(fa, "between", own)[keep], list(own.values()), d[keep], allow_unused=True)
        gr = torch.autograd.grad(_call(R, "between", ref)[keep], list(ref.values()), d[keep].double(),
                                 allow_unused=True)
        for n, a, b in zip(t, go, gr):
            if b is None:
                assert a is None or float(a.abs().max()) == 0.0, n
            else:
                assert rel_l2(a, b) <= TOL[FP32], (keep, n, rel_l2(a, b))


def test_rows_of_constants_and_large_means():
    """A constant row has no deviation: n = 0, not a division by zero. A row far from zero loses the digits
    of its mean over its deviation, 2^10 here: 2^-24 * 2^10 of the normalised values, twice (mean and
    difference)."""
    x = torch.full((1, 3, 256), 5.0, device="cuda")
    z = fa.block_prenorm(x)
    assert float(z.abs().max()) == 0.0
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(1, 50, 256, device="cuda", generator=g) + 1024.0
    assert rel_l2(fa.block_prenorm(x), R.prenorm(x.double())) <= 2.0 ** -13
    x[:, :, 3] = 3e4  # one channel far out of line
    assert rel_l2(fa.block_prenorm(x), R.prenorm(x.double())) <= 2.0 ** -13


def test_nan_and_infinity_stay_in_their_rows():
    t, _ = _make("between", 2, 10, 72, FP32, FP32, "none", seed=7)
    clean = _call(fa, "between", t)
    t["x"][0, 3, 5] = float("nan")
    t["residual"][1, 4, 6] = float("inf")
    got = _call(fa, "between", t)
    keep = torch.ones(2, 10, dtype=torch.bool, device="cuda")
    keep[0, 3] = keep[1, 4] = False
    for a, b in zip(got, clean):
        assert torch.equal(a[keep], b[keep])
    assert bool(torch.isnan(got[0][0, 3]).all()) and bool(torch.isinf(got[0][1, 4, 6]))


def test_strided_inputs_and_gradients():
    t, d = _make("between", 2, 30, 64, BF16, FP32, "all", seed=8)
    want = [a for _, a, _ in _both("between", t, d)]
    s = {k: v.clone() for k, v in t.items()}
    s["x"] = torch.cat((t["x"], t["x"]), -1)[..., :64]
    s["residual"] = t["residual"].transpose(0, 1).contiguous().transpose(0, 1)
    s["gate"] = torch.stack((t["gate"], t["gate"]), -1)[..., 0]
    own = {k: v.detach().requires_grad_(True) for k, v in s.items()}
    out = _call(fa, "between", own)
    d2 = [torch.stack((g, g), -1)[..., 1] for g in d]
    got = (*out, *torch.autograd.grad(out, list(own.values()), d2))
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    u = torch.zeros(t["x"].numel() + 1, device="cuda", dtype=BF16)[1:].view(t["x"].shape)  # an odd address
    u.copy_(t["x"])
    assert rel_l2(fa.block_prenorm(u), R.prenorm(t["x"].double())) <= TOL[BF16]


def test_prenorm_output_dtype():
    t, _ = _make("before", 1, 40, 512, FP32, FP32, "none", seed=9)
    z = fa.block_prenorm(t["x"], t["pre_scale"], t["pre_shift"], out_dtype=BF16)
    ref = fa.block_prenorm(t["x"], t["pre_scale"], t["pre_shift"])
    assert z.dtype == BF16 and torch.equal(z, ref.to(BF16))


def test_equals_adaln_forward():
    """With a gate of ones this is the framework's AdaLN with residual, in the same precision."""
    t, _ = _make("after", 2, 60, 256, BF16, FP32, "all", seed=10, names=("scale", "shift"))
    want = fa.adaptive_layernorm_film_add_residual_forward(t["residual"], t["x"], t["scale"], t["shift"], 1.0,
                                                           output_fp32=True)
    assert rel_l2(fa.block_postnorm_residual(t["residual"], t["x"], t["scale"], t["shift"]), want) <= 1e-6


def test_gradient_matches_differences():
    """Central differences of the float64 definition along each gradient's own direction, h = 1e-4: the
    quotient is good to about 1e-6 of the slope, the gradient to 6e-6."""
    t, d = _make("between", 2, 12, 40, FP32, FP32, "none", seed=11)
    own = {k: v.clone().requires_grad_(True) for k, v in t.items()}
    grads = torch.autograd.grad(_call(fa, "between", own), list(own.values()), d)
    for n, gr in zip(t, grads):
        step = gr.double() / gr.double().norm()
        f = []
        for h in (1e-4, -1e-4):
            p = {k: v.double() for k, v in t.items()}
            p[n] = p[n] + h * step
            f.append(sum(float((o * g.double()).sum()) for o, g in zip(_call(R, "between", p), d)))
        assert abs((f[0] - f[1]) / 2e-4 - float(gr.double().norm())) <= 1e-5 * float(gr.double().norm()), n


def test_empty_and_same_bits():
    t, d = _make("between", 2, 0, 64, BF16, FP32, "none", seed=12)
    for _, a, b in _both("between", t, d):
        assert a.shape == b.shape and (a.numel() == 0 or float(a.abs().max()) == 0.0)
    t, d = _make("between", 0, 5, 64, BF16, FP32, "none", seed=12)
    for _, a, b in _both("between", t, d):
        assert a.shape == b.shape and (a.numel() == 0 or float(a.abs().max()) == 0.0)
    t, d = _make("between", 2, 3001, 512, BF16, FP32, "mixed", seed=13)
    one, two = (_both("between", t, d) for _ in range(2))
    assert all(torch.equal(a, b) for (_, a, _), (_, b, _) in zip(one, two))


def test_captured_step():
    """A step captured twice (workspaces of its own each), replayed on new values. Eager graphs of the
    same leaves are gone by then: torch refuses a capture that meets their gradient nodes."""
    t, d = _make("between", 2, 64, 256, BF16, FP32, "all", seed=14)
    own = {k: v.clone().requires_grad_(True) for k, v in t.items()}

    def step():
        out = _call(fa, "between", own)
        return (*(o.detach() for o in out), *torch.autograd.grad(out, list(own.values()), d))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    with torch.no_grad():
        own["x"].copy_(t["x"] * 2 + 1)
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    want = [a for _, a, _ in _both("between", {**t, "x": t["x"] * 2 + 1}, d)]
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, want))

"""The relative position bias and the block norms together: as a Swin3D block's inference path reads
the bias, and as the sub-layers of a trainable block (norm, window attention, norm + residual + norm, MLP,
norm + residual), whose gradients are compared with the same block in float64."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

import flash_aurora_b200 as fa
import _block_norm_ref as NR
from _rel_bias_ref import attention64
from flash_aurora_b200 import swin3d

pytestmark = pytest.mark.gpu

RES, WS, SS = (4, 12, 24), (2, 6, 12), (1, 3, 6)


def rel_l2(x, ref):
    x, ref = x.detach().double(), ref.detach().double()
    return float((x - ref).norm() / ref.norm().clamp(min=1e-30))


def _block(precision, res, seed=0):
    torch.manual_seed(seed)
    blk = swin3d.Swin3DTransformerBlock(dim=128, num_heads=2, time_dim=64, window_size=WS, shift_size=SS,
                                        precision=precision, rel_pos_bias=True)
    swin3d.init_random_weights_(blk)
    with torch.no_grad():
        blk.attn.relative_position_bias_table.normal_(0.0, 1.0)
    x = torch.randn(2, res[0] * res[1] * res[2], 128, device="cuda")
    c = torch.randn(2, 64, device="cuda")
    return blk.cuda().eval(), x, c


@pytest.mark.parametrize("precision,tol", [("fp32", 2e-5), ("bf16_mixed", 1e-2)])
@pytest.mark.parametrize("res", [RES, (2, 6, 10), (4, 13, 20)])
def test_block_reads_its_bias(precision, tol, res, monkeypatch):
    """The block with its attention replaced by the float64 definition; (2, 6, 10) clamps the window, (4, 13,
    20) pads. Tolerances: the tiers' own, per block output."""
    blk, x, c = _block(precision, res)

    def attention(qkv, heads, table, buckets, *, group_ids, output_layout):
        assert output_layout == "bnc"
        Bw, N, _ = qkv.shape
        q, k, v = qkv.double().view(Bw, N, 3, heads, 64).permute(2, 0, 3, 1, 4)
        out = attention64(q, k, v, table.double(), buckets.index, 0.125, ids=group_ids)
        return out.transpose(1, 2).reshape(Bw, N, heads * 64).to(qkv.dtype)

    with torch.no_grad():
        got = blk(x, c, res)
        monkeypatch.setattr(swin3d, "window_attn_rel_bias_qkvpacked", attention)
        want = blk(x, c, res)
        assert rel_l2(got - x, want - x) <= tol
        blk.attn.relative_position_bias_table.zero_()
        assert rel_l2(blk(x, c, res) - x, want - x) > 10 * tol  # the bias matters


def test_zero_bias_is_the_plain_block():
    blk, x, c = _block("fp32", RES)
    with torch.no_grad():
        blk.attn.relative_position_bias_table.zero_()
        a = blk(x, c, RES)
        blk.attn.relative_position_bias_table = None
        assert rel_l2(a - x, blk(x, c, RES) - x) <= 2e-5


def test_state_dict_gains_only_the_table():
    kw = dict(dim=64, num_heads=1, time_dim=32, window_size=WS)
    plain = set(swin3d.Swin3DTransformerBlock(**kw).state_dict())
    biased = swin3d.Swin3DTransformerBlock(**kw, rel_pos_bias=True).state_dict()
    assert set(biased) - plain == {"attn.relative_position_bias_table"}
    assert biased["attn.relative_position_bias_table"].shape == (3 * 11 * 23, 1)


# ---- a trainable block -------------------------------------------------------------------------
def _partition(x):
    B, D = x.shape[0], x.shape[-1]
    x = torch.roll(x.view(B, *RES, D), (-SS[0], -SS[1], -SS[2]), (1, 2, 3))
    g = [r // w for r, w in zip(RES, WS)]
    x = x.view(B, g[0], WS[0], g[1], WS[1], g[2], WS[2], D).permute(0, 1, 3, 5, 2, 4, 6, 7)
    return x.reshape(-1, 144, D)


def _merge(w, B):
    D = w.shape[-1]
    g = [r // s for r, s in zip(RES, WS)]
    x = w.view(B, *g, *WS, D).permute(0, 1, 4, 2, 5, 3, 6, 7).reshape(B, *RES, D)
    return torch.roll(x, SS, (1, 2, 3)).reshape(B, -1, D)


def _params(D, H, nb, B):
    g = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *s, std=1.0, mean=0.0: torch.randn(*s, device="cuda", generator=g) * std + mean  # noqa: E731
    return {"in_w": rand(D, std=0.1, mean=1.0), "in_b": rand(D, std=0.1), "qkv": rand(3 * D, D, std=D ** -0.5),
            "table": rand(nb, H), "proj": rand(D, D, std=D ** -0.5), "out_w": rand(D, std=0.1, mean=1.0),
            "out_b": rand(D, std=0.1), "gate": rand(B, 1, D, std=0.5, mean=1.0), "alpha": rand(D, std=0.1, mean=1.0),
            "mid_s": rand(B, D, std=0.2), "mid_t": rand(B, D, std=0.2), "fc1": rand(2 * D, D, std=D ** -0.5),
            "fc2": rand(D, 2 * D, std=(2 * D) ** -0.5), "gate2": rand(D, std=0.3, mean=0.5)}


def _step(x, p, H, buckets, ids, ops):
    """One trainable block; ``ops``: prenorm, between, after, attention."""
    prenorm, between, after, attention = ops
    z = prenorm(x, p["in_w"], p["in_b"])
    a = attention(F.linear(_partition(z), p["qkv"]), H, p["table"], buckets, ids)
    a = _merge(F.linear(a, p["proj"]), x.shape[0])
    y, z = between(x, a, p)
    return after(y, F.linear(F.gelu(F.linear(z, p["fc1"])), p["fc2"]), p["gate2"])


OWN = (
    lambda x, w, b: fa.block_prenorm(x, w, b, scale_bias=0.0),
    lambda x, a, p: fa.block_postnorm_residual_prenorm(x, a, p["out_w"], p["out_b"], p["gate"], p["mid_s"], p["mid_t"],
                                                       residual_scale=p["alpha"], scale_bias=0.0),
    lambda y, h, g: fa.block_postnorm_residual(y, h, gate=g, norm="rms"),
    lambda qkv, H, t, b, ids: fa.window_attn_rel_bias_qkvpacked(qkv, H, t, b, group_ids=ids, output_layout="bnc"),
)


def _attention_ref(qkv, H, table, buckets, ids):
    Bw, N, _ = qkv.shape
    q, k, v = qkv.view(Bw, N, 3, H, 64).permute(2, 0, 3, 1, 4)
    return attention64(q, k, v, table, buckets.index, 0.125, ids=ids).transpose(1, 2).reshape(Bw, N, H * 64)


def _between_ref(x, a, p):
    y = NR.postnorm(x, a, p["out_w"], p["out_b"], p["gate"], residual_scale=p["alpha"], scale_bias=0.0)
    return y, NR.prenorm(y, p["mid_s"], p["mid_t"])


REF = (lambda x, w, b: NR.prenorm(x, w, b, scale_bias=0.0), _between_ref,
       lambda y, h, g: NR.postnorm(y, h, gate=g, norm="rms"), _attention_ref)


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.bfloat16, 4e-2)])
def test_training_step(dtype, tol):
    """Loss and gradients of one block. The fp32 tolerance is ten times a single operator's (1e-5), for a chain
    of five of them and four fp32 products; the bf16 one counts roundings: the chain rounds its tensors about
    sixteen times at half a step (2^-9 on average) forward and backward, 16 * 2^-9 = 3.1e-2 if they all add
    up, and the parameters once."""
    B, D, H = 2, 128, 2
    buckets = fa.RelativeBuckets.window(WS, "cuda")
    ids = fa.shifted_window_group_ids(RES, WS, SS, True, torch.device("cuda"))
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(B, RES[0] * RES[1] * RES[2], D, device="cuda", generator=g).to(dtype)
    dout = torch.randn(x.shape, device="cuda", generator=g).to(dtype)
    p = {k: v.to(dtype if k in ("qkv", "proj", "fc1", "fc2") else torch.float32) for k, v in _params(
        D, H, buckets.num_buckets, B).items()}
    own = {k: v.clone().requires_grad_(True) for k, v in {"x": x, **p}.items()}
    ref = {k: v.double().requires_grad_(True) for k, v in {"x": x, **p}.items()}
    prev = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        y = _step(own["x"], own, H, buckets, ids, OWN)
        grads = torch.autograd.grad(y, list(own.values()), dout)
    finally:
        torch.backends.cuda.matmul.allow_tf32 = prev
    yr = _step(ref["x"], ref, H, buckets, ids, REF)
    grads_ref = torch.autograd.grad(yr, list(ref.values()), dout.double())
    assert rel_l2(y, yr) <= tol
    for name, a, b in zip(own, grads, grads_ref):
        assert a.dtype == own[name].dtype and rel_l2(a, b) <= tol, (name, rel_l2(a, b))
    assert fa.device_status() == {"attention": 0, "gemm": 0}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_two_calls_at_once(dtype):
    """Steps on two streams that run at the same time give the bits that they give alone."""
    B, H = 48, 4
    buckets = fa.RelativeBuckets.window(WS, "cuda")
    ids = (torch.arange(144, device="cuda") >= 72).to(torch.uint8).view(1, -1)

    def step(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        qkv = torch.randn(B, 144, 3 * H * 64, device="cuda", generator=g).to(dtype).requires_grad_(True)
        table = torch.randn(buckets.num_buckets, H, device="cuda", generator=g).requires_grad_(True)
        gate = torch.randn(H * 64, device="cuda", generator=g).requires_grad_(True)
        a = fa.window_attn_rel_bias_qkvpacked(qkv, H, table, buckets, group_ids=ids, output_layout="bnc")
        y, z = fa.block_postnorm_residual_prenorm(a.detach(), a, gate=gate)
        return y, z, *torch.autograd.grad((y, z), (qkv, table, gate), (y.detach(), z.detach()))

    alone = [step(s) for s in (0, 1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = step(i)
    torch.cuda.synchronize()
    for a, b in zip(alone, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_captured_block_with_a_bias():
    blk, x, c = _block("bf16_mixed", RES)
    with torch.no_grad():
        want = blk(x, c, RES)
        static = torch.zeros_like(x)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            blk(static, c, RES)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = blk(static, c, RES)
        static.copy_(x)
        graph.replay()
        assert torch.equal(out, want)

"""Cases and plain forms of the trainable Swin block operators: window attention with a learned
relative position bias by buckets, and the norms before / after / between blocks with gate and
residual scale.

``run(state)`` makes the framework's calls when ``own`` is true, and otherwise computes the same
outputs from elementary torch operations in fp32, rounded once at the end.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
HEAD_DIM = 64
EPS = 1e-5


# ----------------------------------------------------------------------------------------------
# Cases
# ----------------------------------------------------------------------------------------------
def _attn(name, train, dtype, windows, heads, window, *, batch=1, masked=False, packed=True, buckets="window"):
    """``windows``: windows per axis of one field; ``window``: tokens per axis of a window."""
    return {"name": name, "op": "attention", "train": train, "dtype": dtype, "batch": batch,
            "g0": windows[0], "g1": windows[1], "g2": windows[2], "w0": window[0], "w1": window[1], "w2": window[2],
            "heads": heads, "masked": masked, "packed": packed, "buckets": buckets}


def _norm(name, train, form, dtype, residual, batch, tokens, dim, *, norm="layer", per_batch=True):
    return {"name": name, "op": "norm", "train": train, "form": form, "dtype": dtype, "residual": residual,
            "batch": batch, "tokens": tokens, "dim": dim, "norm": norm, "per_batch": per_batch}


def listed():
    return [
        # One block of 256 channels on a (4, 36, 72) field, shifted: the smallest serving call.
        _attn("attn_fwd_small", False, "bf16", (2, 6, 6), 4, (2, 6, 12), masked=True),
        # Stage 1 of a quarter-degree field, (4, 180, 360) tokens, 512 channels, shifted: the largest serving call.
        _attn("attn_fwd_stage1", False, "bf16", (2, 30, 30), 8, (2, 6, 12), masked=True),
        # The default (2, 7, 7) window (98 tokens, no multiple of 16), split q / k / v, two fields.
        _attn("attn_fwd_window98", False, "bf16", (2, 8, 8), 6, (2, 7, 7), batch=2, packed=False),
        # The fp32 tier at stage 3's field.
        _attn("attn_fwd_fp32", False, "fp32", (2, 8, 8), 8, (2, 6, 12), masked=True),
        # Training steps: the smallest, stage 1, a ragged window with log-distance buckets, and fp32.
        _attn("attn_train_small", True, "bf16", (2, 6, 6), 4, (2, 6, 12), masked=True),
        _attn("attn_train_stage1", True, "bf16", (2, 30, 30), 8, (2, 6, 12), masked=True),
        _attn("attn_train_log121", True, "bf16", (1, 12, 16), 12, (1, 1, 121), packed=False, buckets="log"),
        _attn("attn_train_fp32", True, "fp32", (2, 8, 8), 8, (2, 6, 12)),
        # Norms: one token's row (latency), stage 1 served, stage 3 trained, an odd width trained in fp32.
        _norm("norm_fwd_one_token", False, "between", "bf16", "fp32", 1, 1, 512),
        _norm("norm_fwd_stage1", False, "between", "bf16", "fp32", 1, 259200, 512),
        _norm("norm_train_stage3", True, "between", "bf16", "fp32", 2, 16200, 2048),
        _norm("norm_train_odd", True, "after", "fp32", "fp32", 3, 7001, 771, norm="rms", per_batch=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.55:
        train = rng.random() < 0.5
        dtype = "fp32" if rng.random() < 0.25 else "bf16"
        buckets = "log" if rng.random() < 0.3 else "window"
        if buckets == "log":
            window = (1, 1, _log_int(rng, 1, 144))
        else:
            w0 = rng.choice((1, 2, 2, 3))
            w1 = rng.randint(1, 8)
            window = (w0, w1, rng.randint(1, max(1, min(18, 144 // (w0 * w1)))))
        heads = rng.choice((1, 2, 3, 4, 5, 6, 8, 12))
        most = 14400 if dtype == "bf16" else 1024
        total = max(1, _log_int(rng, 1, most) // heads)
        g0 = 2 if total >= 8 else 1
        g1 = max(1, int(math.sqrt(total / g0)))
        g2 = max(1, total // (g0 * g1))
        return _attn("", train, dtype, (g0, g1, g2), heads, window, masked=rng.random() < 0.5,
                     packed=rng.random() < 0.5, buckets=buckets) | {"draw": True}
    train = rng.random() < 0.5
    form = rng.choice(("before", "after", "between"))
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    residual = dtype if rng.random() < 0.3 else "fp32"
    dim = _log_int(rng, 8, 4096)
    if rng.random() < 0.7:
        dim = max(8, dim // 8 * 8)
    batch = rng.randint(1, 4)
    tokens = _log_int(rng, 1, max(2, 30_000_000 // (dim * batch)))
    return _norm("", train, form, dtype, residual, batch, tokens, dim, norm=rng.choice(("layer", "rms")),
                 per_batch=rng.random() < 0.5) | {"draw": True}


def _attn_sizes(case):
    nw = case["g0"] * case["g1"] * case["g2"]
    n = case["w0"] * case["w1"] * case["w2"]
    return case["batch"] * nw, nw, case["heads"], n


def work(case):
    if case["op"] == "attention":
        bwin, nw, h, n = _attn_sizes(case)
        e = 2 if case["dtype"] == "bf16" else 4
        tensor = bwin * h * n * HEAD_DIM * e
        table = _num_buckets(case) * h * 4
        side = table + n * n * 4 + (nw * n if case["masked"] else 0)
        flops = 4 * bwin * h * n * n * HEAD_DIM
        if case["train"]:  # q, k, v, dO read, out and dq, dk, dv written
            return {"bytes": 8 * tensor + side + table, "flops": flops + 10 * bwin * h * n * n * HEAD_DIM}
        return {"bytes": 4 * tensor + side, "flops": flops}
    rows = case["batch"] * case["tokens"]
    el = rows * case["dim"]
    e = 2 if case["dtype"] == "bf16" else 4
    r = 2 if case["residual"] == "bf16" else 4
    par = case["dim"] * 4 * (case["batch"] if case["per_batch"] else 1)
    if case["form"] == "before":
        fwd, bwd, npar = el * 2 * e, el * 2 * e, 2
    elif case["form"] == "after":
        fwd, bwd, npar = el * (e + 2 * r), el * (e + 2 * r), 4
    else:
        fwd, bwd, npar = el * (2 * e + 2 * r), el * (2 * e + 2 * r), 6
    if not case["train"]:
        return {"bytes": fwd + npar * par, "flops": el * 12}
    return {"bytes": fwd + bwd + 2 * npar * par, "flops": el * 40}


# ----------------------------------------------------------------------------------------------
# Inputs
# ----------------------------------------------------------------------------------------------
def _num_buckets(case):
    if case["buckets"] == "log":
        return 32
    return (2 * case["w0"] - 1) * (2 * case["w1"] - 1) * (2 * case["w2"] - 1)


def _index(case):
    """(N, N) bucket of each (query, key) pair of a window."""
    if case["buckets"] == "log":
        n = case["w2"]
        rel = torch.arange(n)[None, :] - torch.arange(n)[:, None]  # key - query
        half, exact = 16, 8
        d = rel.abs()
        far = exact + (torch.log(d.clamp(min=1).double() / exact) / math.log(128 / exact) * (half - exact)).long()
        return torch.where(rel > 0, half, 0) + torch.where(d < exact, d, far.clamp(max=half - 1))
    w = (case["w0"], case["w1"], case["w2"])
    grid = torch.stack(torch.meshgrid(*(torch.arange(v) for v in w), indexing="ij")).reshape(3, -1)
    rel = grid[:, :, None] - grid[:, None, :]
    return ((rel[0] + w[0] - 1) * (2 * w[1] - 1) + rel[1] + w[1] - 1) * (2 * w[2] - 1) + rel[2] + w[2] - 1


def _region_ids(case):
    """(nW, N) region ids of half-window shifts: the last window of an axis holds two regions."""
    ids = torch.zeros(1, 1, dtype=torch.long)
    for g, w in (("g0", "w0"), ("g1", "w1"), ("g2", "w2")):
        a = torch.zeros(case[g], case[w], dtype=torch.long)
        a[-1] = torch.where(torch.arange(case[w]) < case[w] - case[w] // 2, 1, 2)
        nw, n = ids.shape
        ids = (ids[:, None, :, None] * 3 + a[None, :, None, :]).reshape(nw * case[g], n * case[w])
    return ids.to(torch.uint8)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def rand(*shape, dtype=torch.float32, std=1.0, mean=0.0):
        return (torch.randn(*shape, device=DEV, generator=gen) * std + mean).to(dtype)

    st = {"case": case}
    if case["op"] == "attention":
        bwin, nw, h, n = _attn_sizes(case)
        if case["packed"]:
            st["qkv"] = rand(bwin, n, 3 * h * HEAD_DIM, dtype=dt)
        else:
            for name in "qkv":
                st[name] = rand(bwin, h, n, HEAD_DIM, dtype=dt)
        st["table"] = rand(_num_buckets(case), h, std=0.5)
        st["index"] = _index(case).to(DEV)
        st["ids"] = _region_ids(case).to(DEV) if case["masked"] else None
        if case["train"]:
            st["dout"] = rand(*((bwin, n, h * HEAD_DIM) if case["packed"] else (bwin, h, n, HEAD_DIM)), dtype=dt)
        if own:
            import flash_aurora_b200 as fa
            st["buckets"] = fa.RelativeBuckets(st["index"], _num_buckets(case))
        leaves = (("qkv",) if case["packed"] else ("q", "k", "v")) + ("table",)
    else:
        b, l, d, form = case["batch"], case["tokens"], case["dim"], case["form"]
        rdt = DTYPES[case["residual"]]
        st["x"] = rand(b, l, d, dtype=dt, std=1.5, mean=0.2)
        par = (b, 1, d) if case["per_batch"] else (d,)
        leaves = ("x",)
        if form != "before":
            st["residual"] = rand(b, l, d, dtype=rdt, std=2.0)
            for name, std in (("post_scale", 0.3), ("post_shift", 0.2), ("gate", 1.0)):
                st[name] = rand(*par, std=std)
            st["residual_scale"] = rand(d, std=0.1, mean=0.8)
            leaves += ("residual", "post_scale", "post_shift", "gate", "residual_scale")
            st["dy"] = rand(b, l, d, dtype=rdt) if case["train"] else None
        if form != "after":
            for name, std in (("pre_scale", 0.3), ("pre_shift", 0.2)):
                st[name] = rand(*par, std=std)
            leaves += ("pre_scale", "pre_shift")
            st["dz"] = rand(b, l, d, dtype=dt) if case["train"] else None
    st["leaves"] = leaves
    if own and case["train"]:
        for name in leaves:
            st[name].requires_grad_(True)
    return st


# ----------------------------------------------------------------------------------------------
# Plain forms: fp32 throughout, each output rounded once
# ----------------------------------------------------------------------------------------------
def _plain_attention(st):
    case = st["case"]
    bwin, nw, h, n = _attn_sizes(case)
    dt = DTYPES[case["dtype"]]
    if case["packed"]:
        q, k, v = st["qkv"].float().reshape(bwin, n, 3, h, HEAD_DIM).permute(2, 0, 3, 1, 4)
    else:
        q, k, v = st["q"].float(), st["k"].float(), st["v"].float()
    scale = 1.0 / math.sqrt(HEAD_DIM)
    x = torch.matmul(q, k.transpose(-1, -2)) * scale
    x = x + st["table"].float()[st["index"]].permute(2, 0, 1)
    if st["ids"] is not None:
        ids = st["ids"]
        mask = (ids[:, :, None] != ids[:, None, :]).float() * -100.0
        x = (x.reshape(bwin // nw, nw, h, n, n) + mask[None, :, None]).reshape(bwin, h, n, n)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    p = x / x.sum(-1, keepdim=True)
    o = torch.matmul(p, v)

    def out_layout(t):
        return t.permute(0, 2, 1, 3).reshape(bwin, n, h * HEAD_DIM) if case["packed"] else t

    out = out_layout(o).to(dt)
    if not case["train"]:
        return out
    do = st["dout"].float()
    if case["packed"]:
        do = do.reshape(bwin, n, h, HEAD_DIM).permute(0, 2, 1, 3)
    dv = torch.matmul(p.transpose(-1, -2), do)
    dp = torch.matmul(do, v.transpose(-1, -2))
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.transpose(-1, -2), q) * scale
    dbias = ds.sum(0).permute(1, 2, 0).reshape(n * n, h)
    dtable = torch.zeros_like(st["table"]).index_add_(0, st["index"].reshape(-1), dbias)
    if case["packed"]:
        dqkv = torch.stack((dq, dk, dv)).permute(1, 3, 0, 2, 4).reshape(bwin, n, 3 * h * HEAD_DIM)
        return out, dqkv.to(dt), dtable
    return out, dq.to(dt), dk.to(dt), dv.to(dt), dtable


def _row_norm(x, kind):
    """Normalised rows and their reciprocal deviation."""
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x * r, r


def _row_norm_grad(dn, n, r, kind):
    g = dn - n * (dn * n).mean(-1, keepdim=True)
    if kind == "layer":
        g = g - dn.mean(-1, keepdim=True)
    return g * r


def _to_param(t, like):
    """Sum of a (B, L, D) gradient over the axes that the parameter is broadcast along."""
    return t.sum(1, keepdim=True) if like.dim() == 3 else t.sum((0, 1))


def _plain_norm(st):
    case, kind = st["case"], st["case"]["norm"]
    form = case["form"]
    x = st["x"].float()
    zdt = DTYPES[case["dtype"]]
    n, r = _row_norm(x, kind)
    if form == "before":
        z = n * (1.0 + st["pre_scale"]) + st["pre_shift"]
        if not case["train"]:
            return z.to(zdt)
        dz = st["dz"].float()
        dx = _row_norm_grad(dz * (1.0 + st["pre_scale"]), n, r, kind)
        return z.to(zdt), dx.to(zdt), _to_param(dz * n, st["pre_scale"]), _to_param(dz, st["pre_shift"])
    res = st["residual"].float()
    p = n * (1.0 + st["post_scale"]) + st["post_shift"]
    y = st["residual_scale"] * res + st["gate"] * p
    ydt = DTYPES[case["residual"]]
    outs = [y.to(ydt)]
    if form == "between":
        m, r2 = _row_norm(y, kind)
        outs.append((m * (1.0 + st["pre_scale"]) + st["pre_shift"]).to(zdt))
    if not case["train"]:
        return outs[0] if form == "after" else tuple(outs)
    dy = st["dy"].float()
    if form == "between":
        dz = st["dz"].float()
        dy = dy + _row_norm_grad(dz * (1.0 + st["pre_scale"]), m, r2, kind)
    dp = dy * st["gate"]
    dx = _row_norm_grad(dp * (1.0 + st["post_scale"]), n, r, kind)
    outs += [dx.to(zdt), (dy * st["residual_scale"]).to(ydt), _to_param(dp * n, st["post_scale"]),
             _to_param(dp, st["post_shift"]), _to_param(dy * p, st["gate"]), (dy * res).sum((0, 1))]
    if form == "between":
        outs += [_to_param(dz * m, st["pre_scale"]), _to_param(dz, st["pre_shift"])]
    return tuple(outs)


# ----------------------------------------------------------------------------------------------
# The framework's calls
# ----------------------------------------------------------------------------------------------
def _own_attention(st):
    import flash_aurora_b200 as fa
    case = st["case"]
    if case["packed"]:
        out = fa.window_attn_rel_bias_qkvpacked(st["qkv"], case["heads"], st["table"], st["buckets"],
                                                group_ids=st["ids"], output_layout="bnc")
    else:
        out = fa.window_attn_rel_bias(st["q"], st["k"], st["v"], st["table"], st["buckets"], group_ids=st["ids"])
    if not case["train"]:
        return out
    grads = torch.autograd.grad(out, [st[name] for name in st["leaves"]], st["dout"])
    return (out.detach(), *grads)


def _own_norm(st):
    import flash_aurora_b200 as fa
    case = st["case"]
    form, kind = case["form"], case["norm"]
    if form == "before":
        outs = (fa.block_prenorm(st["x"], st["pre_scale"], st["pre_shift"], eps=EPS, norm=kind),)
    elif form == "after":
        outs = (fa.block_postnorm_residual(st["residual"], st["x"], st["post_scale"], st["post_shift"], st["gate"],
                                           residual_scale=st["residual_scale"], eps=EPS, norm=kind),)
    else:
        outs = fa.block_postnorm_residual_prenorm(
            st["residual"], st["x"], st["post_scale"], st["post_shift"], st["gate"], st["pre_scale"],
            st["pre_shift"], residual_scale=st["residual_scale"], eps=EPS, norm=kind)
    if not case["train"]:
        return outs if form == "between" else outs[0]
    dout = [st[name] for name in ("dy", "dz") if name in st]
    grads = torch.autograd.grad(outs, [st[name] for name in st["leaves"]], dout)
    return (*(t.detach() for t in outs), *grads)


def run(state):
    if state["case"]["op"] == "attention":
        return _own_attention(state) if own else _plain_attention(state)
    return _own_norm(state) if own else _plain_norm(state)


# ----------------------------------------------------------------------------------------------
# The definition in 64 bits, gradients by differentiation
# ----------------------------------------------------------------------------------------------
def _exact_attention(st):
    case = st["case"]
    bwin, nw, h, n = _attn_sizes(case)
    table = st["table"].detach().double().requires_grad_(True)
    outs, grads = [], []
    step = max(1, 40_000_000 // (h * n * n))
    for a in range(0, bwin, step):
        z = min(bwin, a + step)
        if case["packed"]:
            leaf = [st["qkv"][a:z].detach().double().requires_grad_(True)]
            q, k, v = leaf[0].view(z - a, n, 3, h, HEAD_DIM).unbind(2)
        else:
            leaf = [st[name][a:z].detach().double().requires_grad_(True) for name in "qkv"]
            q, k, v = (t.transpose(1, 2) for t in leaf)
        logits = torch.einsum("bihd,bjhd->bhij", q, k) / 8.0
        logits = logits + torch.einsum("ijh->hij", table[st["index"]])
        if st["ids"] is not None:
            ids = st["ids"][torch.arange(a, z, device=DEV) % nw].long()
            logits = logits - 100.0 * (ids.unsqueeze(2) != ids.unsqueeze(1)).unsqueeze(1)
        w = torch.exp(logits - torch.logsumexp(logits, dim=-1, keepdim=True))
        o = torch.einsum("bhij,bjhd->bihd", w, v)
        o = o.reshape(z - a, n, h * HEAD_DIM) if case["packed"] else o.transpose(1, 2)
        outs.append(o.detach())
        if case["train"]:
            grads.append(torch.autograd.grad(o, leaf + [table], st["dout"][a:z].double()))
    out = torch.cat(outs)
    if not case["train"]:
        return out
    leaves = [torch.cat([g[i] for g in grads]) for i in range(len(grads[0]) - 1)]
    return (out, *leaves, torch.stack([g[-1] for g in grads]).sum(0))


def _exact_norm(st):
    case = st["case"]
    form = case["form"]
    t = {name: st[name].detach().double().requires_grad_(True) for name in st["leaves"]}

    def normed(a):
        if case["norm"] == "layer":
            return (a - a.mean(-1, keepdim=True)) * (a.var(-1, unbiased=False, keepdim=True) + EPS).rsqrt()
        return a * (a.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()

    outs = []
    h = t["x"]
    if form != "before":
        h = t["residual"] * t["residual_scale"] + ((t["post_scale"] + 1.0) * normed(h) + t["post_shift"]) * t["gate"]
        outs.append(h)
    if form != "after":
        outs.append((t["pre_scale"] + 1.0) * normed(h) + t["pre_shift"])
    if not case["train"]:
        outs = [o.detach() for o in outs]
        return tuple(outs) if form == "between" else outs[0]
    dout = [st[name].double() for name in ("dy", "dz") if name in st]
    grads = torch.autograd.grad(outs, [t[name] for name in st["leaves"]], dout)
    return (*(o.detach() for o in outs), *grads)


def exact(case, seed):
    st = prepare(case, seed)
    return _exact_attention(st) if case["op"] == "attention" else _exact_norm(st)

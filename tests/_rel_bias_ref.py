"""Window attention with a relative position bias from its definition, in float64 on any device."""

from __future__ import annotations

import torch


def attention64(q, k, v, table, index, scale, ids=None, mask=None):
    """``q, k, v (Bwin, H, N, Dh)`` float64; ``ids (nW, N)`` or a byte ``mask (nW, N, N)``."""
    Bwin, H, N, _ = q.shape
    x = torch.einsum("whid,whjd->whij", q, k) * scale + table[index.long()].permute(2, 0, 1)
    if ids is not None:
        mask = ids[:, :, None] != ids[:, None, :]
    if mask is not None:
        m = mask.bool()[torch.arange(Bwin, device=q.device) % mask.shape[0]]
        x = x - 100.0 * m[:, None].double()
    return torch.softmax(x, dim=-1) @ v


def reference(q, k, v, table, index, scale, dout, ids=None, mask=None):
    """``(out, dq, dk, dv, dtable)`` in float64, gradients by differentiation."""
    leaves = [t.detach().double().requires_grad_(True) for t in (q, k, v, table)]
    out = attention64(*leaves, index, scale, ids, mask)
    return (out.detach(), *torch.autograd.grad(out, leaves, dout.double()))

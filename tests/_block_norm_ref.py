"""The norms around a residual block from their definitions, in the dtype of the inputs given."""

from __future__ import annotations

import torch


def _rows(p, B):
    """A parameter as (1 or B, 1, D)."""
    return p.reshape(1, 1, -1) if p.ndim == 1 else p.reshape(B, 1, -1)


def normed(x, norm, eps):
    if norm == "layer":
        x = x - x.mean(-1, keepdim=True)
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)


def affine(n, scale, shift, bias):
    B = n.shape[0]
    out = n * (bias if scale is None else bias + _rows(scale, B))
    return out if shift is None else out + _rows(shift, B)


def prenorm(x, scale=None, shift=None, *, scale_bias=1.0, eps=1e-5, norm="layer"):
    return affine(normed(x, norm, eps), scale, shift, scale_bias)


def postnorm(residual, x, scale=None, shift=None, gate=None, *, residual_scale=1.0, scale_bias=1.0, eps=1e-5,
             norm="layer"):
    p = affine(normed(x, norm, eps), scale, shift, scale_bias)
    if gate is not None:
        p = p * _rows(gate, x.shape[0])
    a = _rows(residual_scale, x.shape[0]) if isinstance(residual_scale, torch.Tensor) else residual_scale
    return a * residual + p

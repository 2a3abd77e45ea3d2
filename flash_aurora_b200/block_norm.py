"""The norms before and after a residual block, fused with its gate and residual scale, differentiable.

:mod:`flash_aurora_b200.adaln` is the post-norm of the Swin3D block, forward only. The functions here
cover blocks that are normalised on both sides, and training. With ``N`` the layer norm or the RMS
norm of the last axis, without affine:

* :func:`block_prenorm`                      ``z = N(x) (scale_bias + scale) + shift``
* :func:`block_postnorm_residual`            ``y = residual_scale * residual + gate * (N(x) (scale_bias + scale) + shift)``
* :func:`block_postnorm_residual_prenorm`    that ``y``, and ``z = N(y) (pre_scale_bias + pre_scale) + pre_shift``
  for the next block, in one pass

Tensors are ``(B, L, D)``, float32 or bfloat16, ``D <= 4096``. Scales, shifts, gates and a tensor
``residual_scale`` are ``(D,)`` (learned, shared), ``(B, D)`` or ``(B, 1, D)`` (modulation of a batch element);
``None`` counts as zero for a scale or shift and as one for a gate. With ``scale_bias=0`` a scale is
an ordinary norm weight; with the default of one it is a modulation. Everything is computed in fp32
and each output is rounded once; sums over rows run in a fixed order, so equal calls give equal bits.
Gradients of gradients are not available; forward-mode derivatives and calls inside ``torch.func`` transforms
(``vmap``, ``grad``, ``jvp``) are refused, and ``torch.compile`` is not supported. A step may be captured in a CUDA graph; as for any differentiable
torch call, no eager autograd graph of the same leaves may be alive then (torch refuses such a capture).
"""

from __future__ import annotations

import ctypes
from typing import Optional, Union

import torch

from . import _lib

__all__ = ["block_prenorm", "block_postnorm_residual", "block_postnorm_residual_prenorm"]

_MAX_D = 4096
_DTYPES = (torch.float32, torch.bfloat16)
_NORMS = {"layer": _lib.FA_NORM_LAYER, "rms": _lib.FA_NORM_RMS}
_PARAMS = ("scale", "shift", "gate", "residual_scale", "pre_scale", "pre_shift")


_PTRS, _STRIDES = ctypes.c_void_p * 6, ctypes.c_int64 * 6


class _Call:
    """One call's plain arguments."""

    def __init__(self, form, norm, scale_bias, pre_scale_bias, residual_scale, eps, z_dtype) -> None:
        self.form, self.norm = form, norm
        self.biases = (float(scale_bias), float(pre_scale_bias), residual_scale, float(eps))
        self.z_dtype = z_dtype

    def y_dtype(self, residual) -> torch.dtype:
        return self.z_dtype if self.form == _lib.FA_NORM_BEFORE else residual.dtype


def _ptr(t: Optional[torch.Tensor]):
    return t.data_ptr() if t is not None else None


def _param_args(params, B: int, D: int):
    """fp32 copies where needed, and the C arrays of pointers and batch strides."""
    held = [p if p is None or p.dtype == torch.float32 and p.is_contiguous() else p.to(torch.float32).contiguous()
            for p in params]
    ptrs = _PTRS(*[p if p is None else p.data_ptr() for p in held])
    strides = _STRIDES(*[0 if p is None or p.ndim == 1 else D for p in params])
    return held, ptrs, strides


def _forward(x, residual, params, call: _Call, want_stats: bool):
    B, L, D = x.shape
    dev = x.device
    with _lib.on_device(dev):
        held, ptrs, strides = _param_args(params, B, D)
        y = torch.empty_like(residual) if call.form != _lib.FA_NORM_BEFORE else None
        z = torch.empty(B, L, D, device=dev, dtype=call.z_dtype) if call.form != _lib.FA_NORM_AFTER else None
        stats = torch.empty(B, L, 4, device=dev, dtype=torch.float32) if want_stats else None
        rc = _lib.load().fa_block_norm(
            call.form, call.norm, x.data_ptr(), _lib.dtype_code(x.dtype), _ptr(residual),
            _lib.dtype_code(call.y_dtype(residual)), ptrs, strides, *call.biases, _ptr(y), _ptr(z), _ptr(stats), B, L, D,
            _lib.stream_ptr(dev))
        _lib.check(rc, "block_norm")
    del held
    return y, z, stats


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, call, x, residual, *params):
        y, z, stats = _forward(x, residual, params, call, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, residual, stats, *params)
        ctx.call = call
        if call.form == _lib.FA_NORM_BEFORE:
            return z
        return y if call.form == _lib.FA_NORM_AFTER else (y, z)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        x, residual, stats, *params = ctx.saved_tensors
        call, need = ctx.call, ctx.needs_input_grad
        if all(g is None for g in grads):
            return (None,) * len(need)
        dy = grads[0] if call.form != _lib.FA_NORM_BEFORE else None
        dz = grads[-1] if call.form != _lib.FA_NORM_AFTER else None
        dy, dz = (None if g is None else g.contiguous() for g in (dy, dz))
        B, L, D = x.shape
        dev = x.device
        with _lib.on_device(dev):
            held, ptrs, strides = _param_args(params, B, D)
            dx = torch.empty_like(x) if need[1] else None
            dr = torch.empty_like(residual) if need[2] else None
            dp = [torch.empty(p.shape, device=dev, dtype=torch.float32) if p is not None and n else None
                  for p, n in zip(params, need[3:])]
            lib = _lib.load()
            n = lib.fa_block_norm_workspace(call.form, strides, B, L, D)
            if n < 0:
                _lib.check(int(n), "block_norm backward")
            ws = torch.empty(n, dtype=torch.uint8, device=dev)
            rc = lib.fa_block_norm_backward(
                call.form, call.norm, x.data_ptr(), _lib.dtype_code(x.dtype), _ptr(residual),
                _lib.dtype_code(call.y_dtype(residual)), ptrs, strides, *call.biases, _ptr(dy), _ptr(dz),
                stats.data_ptr(), _ptr(dx), _ptr(dr), _PTRS(*[_ptr(g) for g in dp]), B, L, D,
                ws.data_ptr(), n, _lib.stream_ptr(dev))
            _lib.check(rc, "block_norm backward")
        del held
        return (None, dx, dr, *(g if g is None else g.to(p.dtype) for g, p in zip(dp, params)))


def _check(what: str, x: torch.Tensor, residual: Optional[torch.Tensor], params, norm: str) -> None:
    for t in (x, residual):
        if t is None:
            continue
        if t.device.type != "cuda" or t.dtype not in _DTYPES:
            raise ValueError(f"{what} requires CUDA float32/bfloat16 tensors.")
    if x.ndim != 3:
        raise ValueError(f"{what}: x must be (B, L, D), got {tuple(x.shape)}")
    if residual is not None and (residual.shape != x.shape or residual.device != x.device):
        raise ValueError("residual and x must have the same shape and device.")
    B, _, D = x.shape
    if not 1 <= D <= _MAX_D:
        raise ValueError(f"{what} supports 1 <= D <= {_MAX_D}, got {D}")
    if norm not in _NORMS:
        raise ValueError(f"norm must be 'layer' or 'rms', got {norm!r}")
    for name, p in zip(_PARAMS, params):
        if p is None:
            continue
        if tuple(p.shape) not in ((D,), (B, D), (B, 1, D)):
            raise ValueError(f"{name} must have shape (D,), (B, D) or (B, 1, D) with B, D = {B}, {D}, got {tuple(p.shape)}")
        if p.dtype not in _DTYPES:
            raise ValueError(f"{name} must be float32 or bfloat16")
        if p.device != x.device:
            raise ValueError(f"{name} ({p.device}) must be on {x.device}")


def _run(what, call, x, residual, params, norm):
    _lib.refuse_forward_ad(what, x, residual, *params)
    _check(what, x, residual, params, norm)
    call.norm = _NORMS[norm]
    x = x.contiguous()
    residual = residual.contiguous() if residual is not None else None
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, *params)):
        return _BlockNorm.apply(call, x, residual, *params)
    y, z, _ = _forward(x, residual, params, call, False)
    if call.form == _lib.FA_NORM_BEFORE:
        return z
    return y if call.form == _lib.FA_NORM_AFTER else (y, z)


def _residual_scale(v: Union[float, torch.Tensor]):
    """``(tensor or None, float)`` of a residual scale."""
    return (v, 1.0) if isinstance(v, torch.Tensor) else (None, float(v))


def block_prenorm(
    x: torch.Tensor,
    scale: Optional[torch.Tensor] = None,
    shift: Optional[torch.Tensor] = None,
    *,
    scale_bias: float = 1.0,
    eps: float = 1e-5,
    norm: str = "layer",
    out_dtype: Optional[torch.dtype] = None,
) -> torch.Tensor:
    """``N(x) * (scale_bias + scale) + shift``, the input of a block, in ``out_dtype`` (x's by default)."""
    z_dtype = x.dtype if out_dtype is None else out_dtype
    if z_dtype not in _DTYPES:
        raise ValueError("out_dtype must be float32 or bfloat16")
    call = _Call(_lib.FA_NORM_BEFORE, None, 1.0, scale_bias, 1.0, eps, z_dtype)
    return _run("block_prenorm", call, x, None, (None, None, None, None, scale, shift), norm)


def block_postnorm_residual(
    residual: torch.Tensor,
    x: torch.Tensor,
    scale: Optional[torch.Tensor] = None,
    shift: Optional[torch.Tensor] = None,
    gate: Optional[torch.Tensor] = None,
    *,
    residual_scale: Union[float, torch.Tensor] = 1.0,
    scale_bias: float = 1.0,
    eps: float = 1e-5,
    norm: str = "layer",
) -> torch.Tensor:
    """``residual_scale * residual + gate * (N(x) * (scale_bias + scale) + shift)`` in the residual's dtype,
    for a block's output ``x``."""
    rs, rf = _residual_scale(residual_scale)
    call = _Call(_lib.FA_NORM_AFTER, None, scale_bias, 1.0, rf, eps, x.dtype)
    return _run("block_postnorm_residual", call, x, residual, (scale, shift, gate, rs, None, None), norm)


def block_postnorm_residual_prenorm(
    residual: torch.Tensor,
    x: torch.Tensor,
    scale: Optional[torch.Tensor] = None,
    shift: Optional[torch.Tensor] = None,
    gate: Optional[torch.Tensor] = None,
    pre_scale: Optional[torch.Tensor] = None,
    pre_shift: Optional[torch.Tensor] = None,
    *,
    residual_scale: Union[float, torch.Tensor] = 1.0,
    scale_bias: float = 1.0,
    pre_scale_bias: float = 1.0,
    eps: float = 1e-5,
    norm: str = "layer",
) -> tuple[torch.Tensor, torch.Tensor]:
    """``(y, z)``: :func:`block_postnorm_residual` of one block and :func:`block_prenorm` of its result
    (before rounding) for the next, in one pass. ``y`` has the residual's dtype, ``z`` x's."""
    rs, rf = _residual_scale(residual_scale)
    call = _Call(_lib.FA_NORM_BETWEEN, None, scale_bias, pre_scale_bias, rf, eps, x.dtype)
    return _run("block_postnorm_residual_prenorm", call, x, residual, (scale, shift, gate, rs, pre_scale, pre_shift),
                norm)

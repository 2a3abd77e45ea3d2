"""Window attention with a learned relative position bias by buckets, differentiable.

    out = softmax(q k^T * scale + table[index[i, j], h] + mask) v

beside :mod:`flash_aurora_b200.window_attn`, whose kernels take only the 0 / -100 mask. ``table``
``(num_buckets, H)`` is the learned parameter (the ``relative_position_bias_table`` of Swin models);
:class:`RelativeBuckets` says which bucket each (query, key) pair of a window reads. Gradients reach
q, k, v (or the packed qkv) and the table. Windows hold 1 to 144 tokens, head_dim is 64; masks as in
``window_attn``: region ids or a float bias below -50, each adding -100 to a masked logit. A row whose logits are all
-inf (a bias of -inf for every key) is NaN, as its softmax is.

The tensors' dtype is the tier. bfloat16: logits, softmax and all sums are fp32; the probabilities, and in the
backward pass dS, are rounded to bf16 as operands of the products that follow, so the error against exact arithmetic is
2.1e-3 of the output's norm (2.4e-3 for the gradients) where the output's own rounding makes 1.7e-3. float32: operands
keep 22 bits, or 2^-40 of the largest of their row of 64 if that is more, and sums are fp32: 1.7e-7 and 2.5e-7 of
the norm. The table's gradient is summed in fp32 in both.

A step may be captured in a CUDA graph; as for any differentiable torch call, no eager autograd graph of the same
leaves may be alive then (torch refuses such a capture).

Nothing is kept between calls: the backward pass recomputes the probabilities from q, k, the table
and the row statistics of its own forward call. Sums run in a fixed order, so equal calls give equal
bits. Gradients of gradients are not available; forward-mode derivatives and calls inside ``torch.func``
transforms (``vmap``, ``grad``, ``jvp``) are refused, and ``torch.compile`` is not supported.
"""

from __future__ import annotations

import ctypes
import math
from functools import lru_cache
from typing import Optional

import torch

from . import _lib
from .window_attn import _mask_args

__all__ = ["RelativeBuckets", "window_attn_rel_bias", "window_attn_rel_bias_qkvpacked"]

_MAX_TOKENS = 144
_HEAD_DIM = 64


class RelativeBuckets:
    """The bucket of every (query, key) pair of a window: ``index (N, N)`` integers in
    ``[0, num_buckets)``, with the pairs of each bucket listed for the table's gradient.

    Built once per window shape and device (the range check reads the index on the host). The index
    is copied: changing the given tensor later has no effect. Any stream may use it; a captured graph reads it
    at every replay, so it has to live as long as the graph.
    """

    _stream: Optional[int] = None  # of a GPU's lists: the stream (handle) that their memory belongs to, if known

    def __init__(self, index: torch.Tensor, num_buckets: int, device: Optional[torch.device] = None) -> None:
        if index.ndim != 2 or index.shape[0] != index.shape[1] or not 1 <= index.shape[0] <= _MAX_TOKENS:
            raise ValueError(f"index must be (N, N) with 1 <= N <= {_MAX_TOKENS}, got {tuple(index.shape)}")
        if index.dtype not in (torch.uint8, torch.int16, torch.int32, torch.int64):
            raise ValueError(f"index must hold integers, got {index.dtype}")
        num_buckets = int(num_buckets)
        if not 1 <= num_buckets <= 2 ** 31 - 1:
            raise ValueError(f"num_buckets must be positive, got {num_buckets}")
        dev = index.device if device is None else torch.device(device)
        if dev.type == "cuda" and dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        flat = index.detach().reshape(-1).to(dev, torch.int64)
        lo, hi = torch.stack(torch.aminmax(flat)).tolist()
        if lo < 0 or hi >= num_buckets:
            raise ValueError(f"index holds values outside [0, {num_buckets})")
        values, order = torch.sort(flat, stable=True)
        self.tokens = int(index.shape[0])
        self.num_buckets = num_buckets
        self.device = dev
        self.index = flat.view(self.tokens, self.tokens).to(torch.int32)
        self.order = order.to(torch.int32)
        self.offsets = torch.searchsorted(values, torch.arange(num_buckets + 1, device=dev)).to(torch.int32)
        if dev.type == "cuda":  # ready for every stream from here on
            stream = torch.cuda.current_stream(dev)
            stream.synchronize()
            self._stream = stream.cuda_stream

    def __getstate__(self) -> dict:
        return {**self.__dict__, "_stream": None}  # a copy's memory may belong to another stream

    def _used_by(self, stream: torch.cuda.Stream, *tensors: torch.Tensor) -> None:
        """``stream`` is about to read these tensors: their memory is not given away before it has, even if
        this object is dropped meanwhile."""
        if stream.cuda_stream != self._stream:
            for t in tensors:
                t.record_stream(stream)

    def to(self, device) -> "RelativeBuckets":
        """These buckets on ``device`` (this object if it is there already)."""
        dev = torch.device(device)
        if dev.type == "cuda" and dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        return self if dev == self.device else RelativeBuckets(self.index, self.num_buckets, dev)

    @classmethod
    def window(cls, window_size, device: Optional[torch.device] = None, table_window=None) -> "RelativeBuckets":
        """One bucket per 3-D offset of a ``(wc, wh, ww)`` window, ``(2wc-1)(2wh-1)(2ww-1)`` in all, in
        the order of Swin's ``relative_position_index``. ``table_window``: the buckets are those of this window,
        at least as large on each axis (a window clamped to a small grid reads the table of its full size)."""
        w = tuple(int(v) for v in window_size)
        full = w if table_window is None else tuple(int(v) for v in table_window)
        if len(w) != 3 or len(full) != 3 or min(w) < 1:
            raise ValueError(f"window_size must be three positive integers, got {tuple(window_size)}")
        if any(f < v for f, v in zip(full, w)):
            raise ValueError(f"table_window {full} is smaller than the window {w}")
        pos = torch.cartesian_prod(*(torch.arange(v) for v in w)).view(-1, 3)
        rel = pos[:, None, :] - pos[None, :, :] + torch.tensor([v - 1 for v in full])
        span = [2 * v - 1 for v in full]
        index = (rel[..., 0] * span[1] + rel[..., 1]) * span[2] + rel[..., 2]
        return cls(index, span[0] * span[1] * span[2], device if device is not None else torch.device("cpu"))

    @classmethod
    def log_distance(cls, tokens: int, num_buckets: int = 32, max_distance: int = 128,
                     device: Optional[torch.device] = None) -> "RelativeBuckets":
        """Buckets of the signed distance ``j - i`` along one axis: half of them for keys after the
        query; in each half the distances below ``num_buckets / 4`` have a bucket of their own and the
        rest share logarithmically wider ones up to ``max_distance`` (and beyond)."""
        if num_buckets < 4 or num_buckets % 4 or max_distance <= num_buckets // 4:
            raise ValueError("num_buckets must be a multiple of 4 and max_distance above num_buckets / 4")
        rel = torch.arange(tokens)[None, :] - torch.arange(tokens)[:, None]
        half, exact = num_buckets // 2, num_buckets // 4
        dist = rel.abs()
        far = exact + (torch.log(dist.clamp(min=1).double() / exact) / math.log(max_distance / exact)
                       * (half - exact)).long()
        index = torch.where(dist < exact, dist, far.clamp(max=half - 1)) + torch.where(rel > 0, half, 0)
        return cls(index, num_buckets, device if device is not None else torch.device("cpu"))


def _check_bias(table: torch.Tensor, buckets: RelativeBuckets, H: int, N: int, device: torch.device) -> None:
    if not isinstance(buckets, RelativeBuckets):
        raise TypeError("buckets must be a RelativeBuckets")
    if buckets.tokens != N:
        raise ValueError(f"buckets are of a window of {buckets.tokens} tokens, the tensors hold {N}")
    if tuple(table.shape) != (buckets.num_buckets, H):
        raise ValueError(f"table must have shape (num_buckets, heads) = {(buckets.num_buckets, H)}, "
                         f"got {tuple(table.shape)}")
    if table.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"table must be float32 or bfloat16, got {table.dtype}")
    if table.device != device or buckets.device != device:
        raise ValueError(f"table ({table.device}) and buckets ({buckets.device}) must be on {device}")


def _strided(t: torch.Tensor) -> torch.Tensor:
    """``t (Bwin, H, N, Dh)`` as the kernels can read it: unit head-dim stride, positive strides of
    whole 16-byte units, an aligned base; anything else is copied."""
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t
    unit = 16 // t.element_size()
    if (t.stride(3) == 1 and t.data_ptr() % 16 == 0
            and all(s > 0 and s % unit == 0 or n == 1 for s, n in zip(t.stride()[:3], t.shape[:3]))):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _ptr(t: Optional[torch.Tensor]):
    return t.data_ptr() if t is not None else None


@lru_cache(maxsize=64)
def _bytes(which: str, device: int, *args: int) -> int:
    """Size of a buffer; ``device``, the current one, keeps the cached sizes of unlike devices apart."""
    n = getattr(_lib.load(), "fa_window_attention_rel_bias_" + which)(*args)
    if n < 0:
        _lib.check(int(n), "window_attn_rel_bias")
    return int(n)


# An operand of the kernels: its address and the strides of window, head and token (elements).
def _heads(t: torch.Tensor) -> tuple:
    """``(Bwin, H, N, Dh)``; an axis of one entry gets a legal stride."""
    w, h, n, _ = t.shape
    sw, sh, sn, _ = t.stride()
    return (t.data_ptr(), sw if w > 1 else _HEAD_DIM, sh if h > 1 else _HEAD_DIM, sn if n > 1 else _HEAD_DIM)


def _bnc(t: torch.Tensor) -> tuple:
    """Contiguous ``(Bwin, N, H * Dh)``."""
    return t.data_ptr(), t.shape[1] * t.shape[2], _HEAD_DIM, t.shape[2]


def _qkv(t: torch.Tensor) -> tuple:
    """q, k and v of a contiguous ``(Bwin, N, 3 * H * Dh)``."""
    row = t.shape[2]
    step = row // 3 * t.element_size()
    return tuple((t.data_ptr() + i * step, t.shape[1] * row, _HEAD_DIM, row) for i in range(3))


_STRIDES4, _STRIDES7 = ctypes.c_int64 * 12, ctypes.c_int64 * 21


def _strides(*ops: tuple):
    return (_STRIDES4 if len(ops) == 4 else _STRIDES7)(*[s for o in ops for s in o[1:]])


class _Call:
    """One attention call's arguments besides its tensors. ``kind``: None, "mask_u8" or "group_ids"."""

    def __init__(self, dtype, device, shape, buckets, kind, nW, scale) -> None:
        self.precision = _lib.FA_ATTN_BF16 if dtype == torch.bfloat16 else _lib.FA_ATTN_FP32_3XTF32
        self.device, self.shape, self.buckets, self.kind, self.nW, self.scale = device, shape, buckets, kind, nW, scale

    def masks(self, mask: Optional[torch.Tensor]):
        """The C arguments mask_u8, group_ids, nW, scale."""
        return (_ptr(mask) if self.kind == "mask_u8" else None, _ptr(mask) if self.kind == "group_ids" else None,
                self.nW, self.scale)


def _forward(q, k, v, out, table, mask, call: _Call, want_stats: bool):
    """Launch the forward kernels into the operand ``out``; returns the state that the backward pass reads, with the
    row statistics in it when asked for."""
    Bwin, H, N = call.shape
    dev = call.device
    with _lib.on_device(dev):
        stream = torch.cuda.current_stream(dev)
        call.buckets._used_by(stream, call.buckets.index)
        n = _bytes("state", dev.index, call.precision, H, call.nW if call.kind == "group_ids" else 0)
        at = (n + 15) // 16 * 16  # of the row statistics, in the same buffer
        state = torch.empty(at + Bwin * H * _MAX_TOKENS * 8 if want_stats else n, dtype=torch.uint8, device=dev)
        rc = _lib.load().fa_window_attention_rel_bias(
            call.precision, Bwin, H, N, _HEAD_DIM, q[0], k[0], v[0], out[0], _strides(q, k, v, out), table.data_ptr(),
            _lib.dtype_code(table.dtype), call.buckets.index.data_ptr(), *call.masks(mask), state.data_ptr(),
            state.data_ptr() + at if want_stats else None, stream.cuda_stream)
        _lib.check(rc, "window_attn_rel_bias")
    call.stats_at = at
    return state


def _backward(q, k, v, dout, dq, dk, dv, mask, call: _Call, state, table_dtype) -> Optional[torch.Tensor]:
    """Launch the backward kernels into the operands ``dq``, ``dk``, ``dv``; returns the table's gradient, in
    ``table_dtype`` (None: not asked for)."""
    Bwin, H, N = call.shape
    dev = call.device
    b = call.buckets
    with _lib.on_device(dev):
        stream = torch.cuda.current_stream(dev)
        b._used_by(stream, b.order, b.offsets)
        dtable = None if table_dtype is None else torch.empty(b.num_buckets, H, device=dev, dtype=table_dtype)
        n = _bytes("workspace", dev.index, Bwin, H, N)
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
        rc = _lib.load().fa_window_attention_rel_bias_backward(
            call.precision, Bwin, H, N, _HEAD_DIM, q[0], k[0], v[0], dout[0], dq[0], dk[0], dv[0],
            _strides(q, k, v, dout, dq, dk, dv), *call.masks(mask), state.data_ptr(),
            state.data_ptr() + call.stats_at, b.order.data_ptr(), b.offsets.data_ptr(), b.num_buckets, _ptr(dtable),
            _lib.dtype_code(table_dtype or torch.float32), ws.data_ptr(), n, stream.cuda_stream)
        _lib.check(rc, "window_attn_rel_bias backward")
    return dtable


class _Attn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, mask, call):
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        state = _forward(_heads(q), _heads(k), _heads(v), _heads(out), table, mask, call, True)
        ctx.save_for_backward(q, k, v, mask, state)
        ctx.call, ctx.table_dtype = call, table.dtype
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, mask, state = ctx.saved_tensors
        need = ctx.needs_input_grad
        dout = _strided(dout)
        dq, dk, dv = (torch.empty_like(q, memory_format=torch.contiguous_format) for _ in range(3))
        dtable = _backward(*(_heads(t) for t in (q, k, v, dout, dq, dk, dv)), mask, ctx.call, state,
                           ctx.table_dtype if need[3] else None)
        return dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, dtable, None, None


class _AttnPacked(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, table, mask, call, bnc):
        out, state = _packed_forward(qkv, table, mask, call, bnc, True)
        ctx.save_for_backward(qkv, mask, state)
        ctx.call, ctx.table_dtype, ctx.bnc = call, table.dtype, bnc
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        qkv, mask, state = ctx.saved_tensors
        dqkv = torch.empty_like(qkv)
        if ctx.bnc:
            dout = dout.contiguous()
            dout = dout if dout.data_ptr() % 16 == 0 else dout.clone()
        else:
            dout = _strided(dout)
        dtable = _backward(*_qkv(qkv), _bnc(dout) if ctx.bnc else _heads(dout), *_qkv(dqkv), mask, ctx.call, state,
                           ctx.table_dtype if ctx.needs_input_grad[1] else None)
        return dqkv if ctx.needs_input_grad[0] else None, dtable, None, None, None


def _packed_forward(qkv, table, mask, call, bnc, want_stats):
    Bwin, H, N = call.shape
    shape = (Bwin, N, H * _HEAD_DIM) if bnc else (Bwin, H, N, _HEAD_DIM)
    out = torch.empty(shape, device=qkv.device, dtype=qkv.dtype)
    return out, _forward(*_qkv(qkv), _bnc(out) if bnc else _heads(out), table, mask, call, want_stats)


def _check_window(N: int, Dh: int) -> None:
    if Dh != _HEAD_DIM:
        raise ValueError(f"window attention supports head_dim {_HEAD_DIM}, got {Dh}")
    if not 1 <= N <= _MAX_TOKENS:
        raise ValueError(f"window attention supports 1 to {_MAX_TOKENS} tokens per window, got {N}")


def _check_mask(bias: Optional[torch.Tensor]) -> None:
    if bias is not None and not bias.dtype.is_signed:  # none of its values could be below -50: no mask at all
        raise ValueError(f"bias must hold signed values (masked below -50), got {bias.dtype}")


def _call_args(t, Bwin, H, N, table, buckets, bias, group_ids, scale_qk):
    if bias is not None and group_ids is not None:
        raise ValueError("pass at most one of bias / group_ids")
    _check_bias(table, buckets, H, N, t.device)
    with _lib.on_device(t.device):
        mask_u8, gids, nW, _ = _mask_args(bias, group_ids, t.device, N)
    if (mask_u8 is not None or gids is not None) and nW < 1:
        raise ValueError("a mask needs at least one window")
    scale = 1.0 / math.sqrt(_HEAD_DIM) if scale_qk is None else float(scale_qk)
    if not 1e-30 <= abs(scale) <= 1e30:
        raise ValueError(f"scale_qk must be finite and at least 1e-30 in magnitude, got {scale}")
    kind = "mask_u8" if mask_u8 is not None else "group_ids" if gids is not None else None
    return table.contiguous(), mask_u8 if mask_u8 is not None else gids, _Call(
        t.dtype, t.device, (Bwin, H, N), buckets, kind, nW, scale)


def window_attn_rel_bias(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    table: torch.Tensor,
    buckets: RelativeBuckets,
    bias: Optional[torch.Tensor] = None,
    *,
    scale_qk: Optional[float] = None,
    group_ids: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Attention on ``q, k, v (Bwin, H, N, 64)`` (bfloat16 or float32, one dtype) with the bias
    ``table[buckets.index, h]`` and an optional mask: ``bias (nW, N, N)`` (below -50 means masked, so boolean masks are refused) or
    ``group_ids (nW, N)`` uint8. Window ``b`` reads mask ``b % nW``. Returns ``(Bwin, H, N, 64)``."""
    _lib.refuse_forward_ad("window_attn_rel_bias", q, k, v, table)
    if q.ndim != 4 or q.shape != k.shape or q.shape != v.shape:
        raise ValueError("q, k, v must all be (Bwin, H, N, Dh)")
    if q.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"window_attn_rel_bias supports bfloat16 and float32; got {q.dtype}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v must share a dtype")
    Bwin, H, N, Dh = q.shape
    _check_window(N, Dh)
    if H < 1:
        raise ValueError("at least one head is needed")
    _check_mask(bias)
    if not q.is_cuda:
        raise RuntimeError("B200 window attention requires CUDA tensors.")
    if k.device != q.device or v.device != q.device:
        raise ValueError("q, k and v must be on one device")
    table, mask, call = _call_args(q, Bwin, H, N, table, buckets, bias, group_ids, scale_qk)
    q, k, v = _strided(q), _strided(k), _strided(v)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, table)):
        return _Attn.apply(q, k, v, table, mask, call)
    out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    _forward(_heads(q), _heads(k), _heads(v), _heads(out), table, mask, call, False)
    return out


def window_attn_rel_bias_qkvpacked(
    qkv: torch.Tensor,
    num_heads: int,
    table: torch.Tensor,
    buckets: RelativeBuckets,
    bias: Optional[torch.Tensor] = None,
    *,
    scale_qk: Optional[float] = None,
    output_layout: str = "bhnd",
    group_ids: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """:func:`window_attn_rel_bias` on the packed ``Linear(D, 3D)`` output ``(Bwin, N, 3 * H * 64)``,
    contiguous. Returns ``(Bwin, H, N, 64)``, or ``(Bwin, N, H * 64)`` with ``output_layout="bnc"``."""
    _lib.refuse_forward_ad("window_attn_rel_bias_qkvpacked", qkv, table)
    if qkv.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"qkv-packed path supports bfloat16 and float32; got {qkv.dtype}")
    if qkv.ndim != 3:
        raise ValueError(f"qkv must have shape (Bwin, N, 3*C); got {tuple(qkv.shape)}")
    if not qkv.is_contiguous():
        raise ValueError("qkv-packed path requires contiguous qkv linear output")
    if num_heads < 1 or qkv.shape[-1] % (3 * num_heads) != 0:
        raise ValueError(f"last dim {qkv.shape[-1]} must be divisible by 3*num_heads={3 * num_heads}")
    if output_layout not in {"bhnd", "bnc"}:
        raise ValueError(f"output_layout must be 'bhnd' or 'bnc', got {output_layout!r}")
    Bwin, N, three_c = qkv.shape
    H = int(num_heads)
    _check_window(N, three_c // (3 * H))
    _check_mask(bias)
    if not qkv.is_cuda:
        raise RuntimeError("B200 window attention requires CUDA tensors.")
    table, mask, call = _call_args(qkv, Bwin, H, N, table, buckets, bias, group_ids, scale_qk)
    if qkv.data_ptr() % 16:
        qkv = qkv.clone()
    bnc = output_layout == "bnc"
    if torch.is_grad_enabled() and (qkv.requires_grad or table.requires_grad):
        return _AttnPacked.apply(qkv, table, mask, call, bnc)
    return _packed_forward(qkv, table, mask, call, bnc, False)[0]

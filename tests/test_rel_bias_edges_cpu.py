"""Host-side edges of window attention with a relative position bias (no GPU needed)."""

from __future__ import annotations

import copy
import ctypes
import pickle
from types import SimpleNamespace

import pytest
import torch
from torch.autograd import forward_ad

import flash_aurora_b200 as fa
from flash_aurora_b200 import _lib

P = ctypes.c_void_p(1 << 20)
STRIDES = (ctypes.c_int64 * 21)(*([64] * 21))


def _backward(workspace, nbytes, Bwin=4, dtable=P):
    return _lib.load().fa_window_attention_rel_bias_backward(
        0, Bwin, 2, 16, 64, P, P, P, P, P, P, P, STRIDES, None, None, 0, 0.125, P, P, P, P, 5, dtable, 0, workspace,
        nbytes, None)


def test_workspace_must_be_aligned():
    """The partial bias gradients in it are written 16 bytes at a time."""
    lib = _lib.load()
    for off in (2, 4, 8):
        assert _backward(ctypes.c_void_p((1 << 20) + off), 1 << 40) == _lib.FA_ERR_INVALID
        assert b"workspace" in lib.fa_last_error() and b"16-byte aligned" in lib.fa_last_error()


def test_workspace_size_is_exact():
    """One 144 x 144 fp32 partial per block and head that meet: 8 blocks of one tile each, and 2 heads."""
    lib = _lib.load()
    need = (8 + 2) * 144 * 144 * 4
    assert lib.fa_window_attention_rel_bias_workspace(4, 2, 16) == need
    assert _backward(P, need - 1) == _lib.FA_ERR_INVALID and b"workspace" in lib.fa_last_error()


class _Recorded:
    def __init__(self):
        self.streams = []

    def record_stream(self, s):
        self.streams.append(s)


def test_buckets_are_recorded_with_other_streams():
    """Only a stream other than the one that the lists' memory belongs to has to be recorded; of a copy the
    owner is unknown, so every stream is."""
    b = fa.RelativeBuckets.window((1, 2, 3))
    own, other = SimpleNamespace(cuda_stream=16), SimpleNamespace(cuda_stream=32)
    b._stream = 16
    t, u = _Recorded(), _Recorded()
    b._used_by(own, t, u)
    assert t.streams == u.streams == []
    b._used_by(other, t, u)
    assert t.streams == u.streams == [other]
    for c in (copy.copy(b), copy.deepcopy(b), pickle.loads(pickle.dumps(b))):
        assert torch.equal(c.index, b.index) and c.num_buckets == b.num_buckets
        t = _Recorded()
        c._used_by(own, t)
        assert t.streams == [own]


def test_forward_mode_is_refused():
    """A dual tensor's tangent would be lost; its primal alone goes on to the next check (CPU tensors)."""
    b = fa.RelativeBuckets.window((1, 2, 4))
    table, q, qkv = torch.zeros(b.num_buckets, 2), torch.zeros(3, 2, 8, 64), torch.zeros(3, 8, 384)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for i in range(4):
            args = [dual(t) if i == j else t for j, t in enumerate((q, q, q, table))]
            with pytest.raises(NotImplementedError, match="forward-mode"):
                fa.window_attn_rel_bias(*args, b)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            fa.window_attn_rel_bias_qkvpacked(dual(qkv), 2, table, b)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            fa.window_attn_rel_bias_qkvpacked(qkv, 2, dual(table), b)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            fa.window_attn_rel_bias(dual(q), q, q, table, b)
        with pytest.raises(RuntimeError, match="CUDA"):
            fa.window_attn_rel_bias(q, q, q, table, b)


@pytest.mark.parametrize("dtype", [torch.bool, torch.uint8])
def test_masks_that_cannot_mask_are_refused(dtype):
    """A boolean mask is never below -50: it would be taken for "nothing masked"."""
    b = fa.RelativeBuckets.window((1, 2, 4))
    table, q = torch.zeros(b.num_buckets, 2), torch.zeros(3, 2, 8, 64)
    mask = torch.ones(1, 8, 8, dtype=dtype)
    with pytest.raises(ValueError, match="signed"):
        fa.window_attn_rel_bias(q, q, q, table, b, mask)
    with pytest.raises(ValueError, match="signed"):
        fa.window_attn_rel_bias_qkvpacked(torch.zeros(3, 8, 384), 2, table, b, bias=mask)
    with pytest.raises(RuntimeError, match="CUDA"):
        fa.window_attn_rel_bias(q, q, q, table, b, mask.float())


def test_buckets_pickled_without_a_stream():
    """A pickle of the first version's object has no stream: unknown, so every stream is recorded."""
    b = fa.RelativeBuckets.window((1, 2, 3))
    b.__dict__.pop("_stream", None)
    t, s = _Recorded(), SimpleNamespace(cuda_stream=0)
    b._used_by(s, t)
    assert t.streams == [s]

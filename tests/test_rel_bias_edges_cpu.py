"""Host-side edges of window attention with a relative position bias (no GPU needed)."""

from __future__ import annotations

import ctypes

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

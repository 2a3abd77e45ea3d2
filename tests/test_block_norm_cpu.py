"""Refusals of the block norms that need no GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

import flash_aurora_b200 as fa


def test_refusals_before_any_launch():
    x = torch.zeros(2, 3, 8)
    with pytest.raises(ValueError, match="CUDA"):
        fa.block_prenorm(x)
    with pytest.raises(ValueError, match="CUDA"):
        fa.block_postnorm_residual(x, x)
    with pytest.raises(ValueError, match="CUDA"):
        fa.block_postnorm_residual_prenorm(x, x)
    with pytest.raises(ValueError, match="out_dtype"):
        fa.block_prenorm(x, out_dtype=torch.float16)


def test_argument_checks():
    from flash_aurora_b200.block_norm import _check
    x = torch.zeros(2, 3, 8, device="meta")

    class Cuda:  # the checks read only these
        def __init__(self, *shape, dtype=torch.float32, device=torch.device("cuda", 0)):
            self.shape, self.dtype, self.device, self.ndim = torch.Size(shape), dtype, device, len(shape)

    x = Cuda(2, 3, 8)
    none = (None,) * 6
    _check("op", x, None, none, "layer")
    _check("op", x, x, (Cuda(8), Cuda(2, 8), Cuda(2, 1, 8), None, None, None), "rms")
    with pytest.raises(ValueError, match="float32/bfloat16"):
        _check("op", Cuda(2, 3, 8, dtype=torch.float16), None, none, "layer")
    with pytest.raises(ValueError, match=r"\(B, L, D\)"):
        _check("op", Cuda(3, 8), None, none, "layer")
    with pytest.raises(ValueError, match="same shape"):
        _check("op", x, Cuda(2, 3, 9), none, "layer")
    with pytest.raises(ValueError, match="4096"):
        _check("op", Cuda(1, 1, 4097), None, none, "layer")
    with pytest.raises(ValueError, match="4096"):
        _check("op", Cuda(1, 1, 0), None, none, "layer")
    with pytest.raises(ValueError, match="'layer' or 'rms'"):
        _check("op", x, None, none, "group")
    with pytest.raises(ValueError, match="gate must have shape"):
        _check("op", x, x, (None, None, Cuda(2, 3, 8), None, None, None), "layer")
    with pytest.raises(ValueError, match="shift must be float32 or bfloat16"):
        _check("op", x, x, (None, Cuda(8, dtype=torch.float64), None, None, None, None), "layer")
    with pytest.raises(ValueError, match="must be on"):
        _check("op", x, x, (Cuda(8, device=torch.device("cpu")), None, None, None, None, None), "layer")


def test_abi_refusals_without_a_gpu():
    from flash_aurora_b200 import _lib
    lib = _lib.load()
    p = ctypes.c_void_p(1 << 20)
    none = (ctypes.c_void_p * 6)()
    zero = (ctypes.c_int64 * 6)()

    def fwd(form=2, norm=0, x=p, xd=1, r=p, yd=0, params=none, strides=zero, y=p, z=p, stats=None, B=1, L=4, D=64):
        return lib.fa_block_norm(form, norm, x, xd, r, yd, params, strides, 1.0, 1.0, 1.0, 1e-5, y, z, stats, B, L, D,
                                 None)

    assert fwd(form=3) == _lib.FA_ERR_INVALID and b"form" in lib.fa_last_error()
    assert fwd(norm=2) == _lib.FA_ERR_INVALID and b"norm" in lib.fa_last_error()
    assert fwd(xd=2) == _lib.FA_ERR_INVALID and b"dtype" in lib.fa_last_error()
    assert fwd(yd=5) == _lib.FA_ERR_INVALID
    assert fwd(D=4097) == _lib.FA_ERR_UNSUPPORTED and b"4096" in lib.fa_last_error()
    assert fwd(D=0) == _lib.FA_ERR_INVALID and fwd(L=-1) == _lib.FA_ERR_INVALID
    assert fwd(B=1 << 30, L=1 << 40) == _lib.FA_ERR_INVALID and b"too large" in lib.fa_last_error()
    assert fwd(x=None) == _lib.FA_ERR_INVALID and fwd(r=None) == _lib.FA_ERR_INVALID
    assert fwd(y=None) == _lib.FA_ERR_INVALID and fwd(z=None) == _lib.FA_ERR_INVALID
    assert fwd(stats=ctypes.c_void_p(8)) == _lib.FA_ERR_INVALID and b"stats" in lib.fa_last_error()
    assert fwd(strides=(ctypes.c_int64 * 6)(64)) == _lib.FA_ERR_INVALID  # a stride without its parameter
    assert fwd(B=0) == _lib.FA_OK and fwd(L=0, x=None) == _lib.FA_OK
    n = lib.fa_block_norm_workspace(2, zero, 1, 4, 64)
    assert n > 0 and n % (6 * 64 * 4) == 0
    assert lib.fa_block_norm_workspace(2, zero, 1, 4, 4097) == _lib.FA_ERR_INVALID

    def bwd(stats=p, dparams=none, ws=p, nbytes=1 << 30):
        return lib.fa_block_norm_backward(2, 0, p, 1, p, 0, none, zero, 1.0, 1.0, 1.0, 1e-5, p, p, stats, p, p, dparams,
                                          1, 4, 64, ws, nbytes, None)

    assert bwd(stats=None) == _lib.FA_ERR_INVALID and b"stats" in lib.fa_last_error()
    assert bwd(dparams=None) == _lib.FA_ERR_INVALID
    assert bwd(ws=None) == _lib.FA_ERR_INVALID and b"workspace" in lib.fa_last_error()
    assert bwd(nbytes=8) == _lib.FA_ERR_INVALID

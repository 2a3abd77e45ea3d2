"""Host-side edges of the block norms (no GPU needed)."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import flash_aurora_b200 as fa


def test_forward_mode_is_refused():
    """A dual tensor's tangent would be lost, whichever operand carries it."""
    x, p = torch.zeros(2, 3, 8), torch.zeros(8)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        with pytest.raises(NotImplementedError, match="forward-mode"):
            fa.block_prenorm(dual(x))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            fa.block_prenorm(x, shift=dual(p))
        for i in range(2):
            pair = [dual(x) if i == j else x for j in range(2)]
            with pytest.raises(NotImplementedError, match="forward-mode"):
                fa.block_postnorm_residual(*pair)
        for name in ("scale", "shift", "gate", "residual_scale", "pre_scale", "pre_shift"):
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                fa.block_postnorm_residual_prenorm(x, x, **{name: dual(p)})
        with pytest.raises(ValueError, match="CUDA"):
            fa.block_prenorm(x)

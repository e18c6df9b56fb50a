"""Corners of the gated residual trunk's Python surface that need no GPU."""

from __future__ import annotations

import pytest
import torch

import fused_hoad


def test_forward_mode_is_refused_on_the_host():
    import torch.autograd.forward_ad as forward

    x = torch.zeros(2, 4)
    with forward.dual_level():
        dual = forward.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward-mode"):
            fused_hoad.gated_feed_forward(dual, x, x, x)
        with pytest.raises(RuntimeError, match="forward-mode"):
            fused_hoad.residual_norm(x, dual, x[0])
        with pytest.raises(RuntimeError, match="forward-mode"):
            fused_hoad.rms_norm(dual, x[0])

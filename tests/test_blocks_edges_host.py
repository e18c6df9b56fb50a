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


def test_trunk_keeps_its_scales_in_float32():
    """The residual scales' steps are smaller than bfloat16's near 1."""
    trunk = fused_hoad.GatedResidualTrunk(2, 8, 16, 3)
    value = 1 + 2.0**-12
    with torch.no_grad():
        for s in trunk.scale:
            s.fill_(value)
    for cast in (lambda t: t.bfloat16(), lambda t: t.to(torch.bfloat16), lambda t: t.half(),
                 lambda t: t.double(), lambda t: t.float()):
        cast(trunk)
        assert all(s.dtype == torch.float32 and float(s) == value and s.requires_grad for s in trunk.scale)
    assert {p.dtype for n, p in trunk.bfloat16().named_parameters() if not n.startswith("scale")} == {torch.bfloat16}
    assert len(list(trunk.scale)) == 3 and {n for n, _ in trunk.named_parameters()} >= {"scale.0", "scale.2"}
    moved = fused_hoad.GatedResidualTrunk(2, 8, 16, 3).to("meta")
    assert moved.scale[0].device.type == "meta" and moved.scale[0].dtype == torch.float32

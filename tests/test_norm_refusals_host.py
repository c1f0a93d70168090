"""CPU-only checks of what the norms' differentiable forms refuse, before a device is looked for."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD


@pytest.mark.parametrize("which", ["x", "weight", "bias"])
@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_is_refused(built_lib, which, requires_grad):
    """A tangent would be lost without a word."""
    from unirl_amd import models

    with fwAD.dual_level():
        t = {"x": torch.randn(3, 8), "weight": torch.ones(8), "bias": torch.zeros(8)}
        t[which] = fwAD.make_dual(t[which].requires_grad_(requires_grad), torch.ones_like(t[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            models.layer_norm(t["x"], t["weight"], t["bias"])
        if which != "bias":
            with pytest.raises(RuntimeError, match="forward-mode"):
                models.rms_norm(t["x"], t["weight"])
        with pytest.raises(RuntimeError, match="forward-mode"):
            models.modulated_layer_norm(t["x"], *(t[k].expand(3, 8) for k in ("weight", "bias")))

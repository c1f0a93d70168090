"""CPU-only checks of what the norms' differentiable forms refuse, before a device is looked for."""

import ctypes

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


def test_the_limit_of_groups_is_that_of_the_parameters_gradients(built_lib):
    """With nothing to compute the call returns before it launches: only the order of its checks is looked at."""
    from unirl_amd import _native as N

    fake = 0x10000  # never dereferenced
    desc = N.NormDesc(x=fake, dtype=N.BF16, x_group_stride=64, x_row_stride=64, groups=65536, rows=1, D=64, gain=fake, gain_dtype=N.BF16,
                      gain_group_stride=64, center=1, eps=1e-5, mean=fake, rstd=fake)
    call = lambda dgain: N.lib().unirl_layer_norm_bwd(ctypes.byref(desc), fake, 64, 64, None, dgain, None, 1, fake, 1 << 40, None)
    assert call(None) == 0 and call(fake) == -6

"""The norm over more groups than one launch takes: modulation per token."""

import pytest
import torch

from tests.test_gpu_norm import check, make, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [8, 33, 264])
def test_gradient_of_the_rows_over_many_groups(dev, D):
    """dx alone has no limit of groups."""
    from unirl_amd import models

    x, w, b, dy = make((70001, 1, D), torch.float32, D, True)
    want = reference(x, w, b, dy, 1e-5, False, 1.0)
    X = x.to(dev).requires_grad_(True)
    y = models.modulated_layer_norm(X, w.to(dev), b.to(dev), 1e-5)
    (dx,) = torch.autograd.grad(y, X, dy.to(dev))
    check(y, want["y"], "y")
    check(dx, want["dx"], "dx")


def test_too_many_groups_for_the_gains_gradient_are_refused_in_the_forward(dev):
    from unirl_amd import models

    x = torch.randn(65536, 1, 8, device=dev)
    w, b = torch.randn(65536, 8, device=dev), torch.randn(65536, 8, device=dev)
    for which in (w, b):
        which.requires_grad_(True)
        with pytest.raises(ValueError, match="limit of 65535"):
            models.modulated_layer_norm(x, w, b)
        with torch.no_grad():
            models.modulated_layer_norm(x, w, b)
        which.requires_grad_(False)
    x, w, b = x[:65535], w[:65535].requires_grad_(True), b[:65535].requires_grad_(True)
    dw, db = torch.autograd.grad(models.modulated_layer_norm(x, w, b).sum(), (w, b))
    want = reference(x.cpu(), w.detach().cpu(), b.detach().cpu(), torch.ones(65535, 1, 8), 1e-6, False, 1.0)
    check(dw, want["dw"], "dw")
    check(db, want["db"], "db")

"""Norms in front of a policy's output, forward and backward as fused kernels.

* ``rms_norm`` / ``layer_norm`` -- the final norm of an AR policy, whose output the head reads (the
  ``hidden`` that ``unirl/models/qwen3/ar.py:82-99`` hands to ``lm_head``);
  ``chunked_replay_logp(final_norm=...)`` applies it.
* ``modulated_layer_norm`` -- the norm with a scale and a shift per sample in front of a diffusion
  policy's output projection (the velocities that ``unirl/models/sd3/diffusion.py:467-497`` replays).

The forward keeps the row's mean and reciprocal deviation (8 bytes a row) for the backward, which
reads ``x`` and ``dy`` once and sums the gain's and bias's gradients in the same pass.  Forward and
backward are one C++ autograd node (``csrc/torch_host.cpp``); the backward is not differentiable and
there is no forward-mode derivative (both raise).  A backward can be captured into a graph, but not for a
leaf over which a graph built on the default stream is still alive: that is refused.
"""

from __future__ import annotations

from typing import Optional

import torch

from .. import _native as N


def layer_norm(
    x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5
) -> torch.Tensor:
    """Layer norm over the last dimension with an optional gain and bias ``[D]``, in ``x``'s dtype
    (computed in fp32, rounded once); differentiable in ``x``, ``weight`` and ``bias``."""
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None and p.dim() != 1:
            raise ValueError(f"{name} must be [D]; got {tuple(p.shape)} (modulated_layer_norm takes one row per sample)")
    return N.host().norm(x, weight, bias, eps, False, False)


def rms_norm(
    x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-6, *, unit_offset: bool = False
) -> torch.Tensor:
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last dimension (``* (1 + weight)`` with
    ``unit_offset``), in ``x``'s dtype (computed in fp32, rounded once: the product with the gain is
    not preceded by a rounding to 16 bits); differentiable in ``x`` and ``weight``."""
    if weight is not None and weight.dim() != 1:
        raise ValueError(f"weight must be [D]; got {tuple(weight.shape)}")
    return N.host().norm(x, weight, None, eps, True, unit_offset)


def modulated_layer_norm(x: torch.Tensor, scale: torch.Tensor, shift: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """``layer_norm(x[b]) * (1 + scale[b]) + shift[b]`` for ``x [B, ..., D]`` and ``scale``, ``shift`` ``[B, D]``
    (or ``[B, 1, ..., D]``; halves of one projection's output are read in place), in ``x``'s dtype;
    differentiable in all three, the modulation's gradients summed over each sample's rows (for at most 65535
    samples)."""
    if x.dim() < 2:
        raise ValueError(f"x must be [B, ..., D]; got {tuple(x.shape)}")
    rows = (x.shape[0], x.shape[-1])
    given = {"scale": scale, "shift": shift}
    for name, p in given.items():
        if p.dim() < 2 or (p.shape[0], p.shape[-1]) != rows or p.numel() != rows[0] * rows[1]:
            raise ValueError(f"{name} must be [{rows[0]}, {rows[1]}]; got {tuple(p.shape)}")
        given[name] = p if p.dim() == 2 else p.reshape(rows)
    return N.host().norm(x, given["scale"], given["shift"], eps, False, True)


__all__ = ["layer_norm", "modulated_layer_norm", "rms_norm"]

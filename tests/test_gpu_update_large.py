"""Norm, gradient norm and AdamW past 2^31 elements: a call on the whole against one on its tail alone, and a
sum that is known exactly."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BIG = (1 << 31) + (1 << 22)


def test_norm_rows_past_2g_elements(dev):
    from unirl_amd import ops

    D = 2048
    rows = BIG // D
    x = torch.empty(rows, D, dtype=torch.bfloat16, device=dev).normal_()
    w = torch.rand(D, device=dev).bfloat16()
    y, _, rstd = ops.layer_norm(x, w, rms=True, want_stats=True)
    tail = ops.layer_norm(x[-5:].clone(), w, rms=True, want_stats=True)
    assert torch.equal(y[-5:], tail[0]) and torch.equal(rstd[-5:], tail[2])
    dx, dw, _ = ops.layer_norm_bwd(y, x, None, rstd, w, rms=True)
    dx_tail, _, _ = ops.layer_norm_bwd(y[-5:].clone(), x[-5:].clone(), None, rstd[-5:], w, rms=True)
    assert torch.equal(dx[-5:], dx_tail) and bool(torch.isfinite(dw).all())


def test_narrow_rows_past_2g_elements(dev):
    from unirl_amd import ops

    D = 128
    x = torch.empty(BIG // D, D, dtype=torch.bfloat16, device=dev).normal_()
    w, b = torch.rand(D, device=dev).bfloat16(), torch.rand(D, device=dev).bfloat16()
    y, mean, rstd = ops.layer_norm(x, w, b, want_stats=True)
    tail = ops.layer_norm(x[-7:].clone(), w, b)
    assert torch.equal(y[-7:], tail[0])
    dx, _, _ = ops.layer_norm_bwd(y, x, mean, rstd, w, b)
    dx_tail, _, _ = ops.layer_norm_bwd(y[-7:].clone(), x[-7:].clone(), mean[-7:], rstd[-7:], w, b)
    assert torch.equal(dx[-7:], dx_tail)


def test_grad_norm_past_2g_elements(dev):
    from unirl_amd import ops

    g = torch.full((BIG,), 0.5, dtype=torch.bfloat16, device=dev)
    g[-1] = 2.0**16  # counts only when the last element is read
    exact = math.sqrt(0.25 * (BIG - 1) + 2.0**32)
    assert abs(float(ops.grad_norm([g])) / exact - 1) <= 1.01 * 2.0**-24


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_past_2g_elements(dev, bits):
    from unirl_amd import ops

    n, cut = BIG + 77, BIG - 4096  # a multiple of 256 in front of the tail
    p = torch.full((n,), 1.0, dtype=torch.bfloat16, device=dev)
    g = torch.empty(n, dtype=torch.bfloat16, device=dev).normal_()
    dtype = torch.float32 if bits == 32 else torch.uint8
    m, v = torch.zeros(n, dtype=dtype, device=dev), torch.zeros(n, dtype=dtype, device=dev)
    kw, tail_kw = {}, {}
    if bits == 8:
        ms, vs = (torch.zeros(-(-n // 256), dtype=torch.uint8, device=dev) for _ in range(2))
        kw = dict(exp_avg_scales=[ms], exp_avg_sq_scales=[vs], index_bases=[0])
        tail_kw = dict(exp_avg_scales=[ms[cut // 256 :].clone()], exp_avg_sq_scales=[vs[cut // 256 :].clone()], index_bases=[cut])
    tail = [t[cut:].clone() for t in (p, g, m, v)]
    hyper = dict(lr=0.1, step=1, seed=3)
    ops.adamw_step([p], [g], [m], [v], **hyper, **kw)
    ops.adamw_step(*[[t] for t in tail], **hyper, **tail_kw)
    for whole, part in zip((p, m, v), (tail[0], tail[2], tail[3])):
        assert torch.equal(whole[cut:], part)
    if bits == 8:
        assert torch.equal(ms[cut // 256 :], tail_kw["exp_avg_scales"][0])
        a, b = ops.adamw_moments(m, v, ms, vs, dtype=torch.bfloat16)
        c, d = ops.adamw_moments(tail[2], tail[3], tail_kw["exp_avg_scales"][0], tail_kw["exp_avg_sq_scales"][0],
                                 dtype=torch.bfloat16)
        assert torch.equal(a[cut:], c) and torch.equal(b[cut:], d)
    assert bool((p != 1.0).float().mean() > 0.99)

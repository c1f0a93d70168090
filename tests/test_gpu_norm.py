"""Layer norm / RMS norm / modulated layer norm, forward and backward, against 64-bit formulas.

Tolerances, with u = 2^-24 (half a unit of fp32) and h(T) = finfo(T).eps / 2:

* A sum over a row adds each term through at most 32 (lane) + 6 (wavefront) + 16 (workgroup) = 54
  additions, so |error| <= 54 u sum|terms|; with the product by the rounded 1/D the mean is off by at
  most 57 u A, A = mean|x| (layer norm; the RMS norm has no mean).
* The centred values are off by that and u |x - mu|.  The variance is then off by at most
  2 * 57 u A s + 60 u relative (s = rstd), the root by half of it and 5 u for the sum with eps, the root and the
  division: r = 57 u A s + 35 u relative.
* xh = (x - mu) s:  e = 57 u A s + |xh| (57 u A s + 40 u);  y: |w| e + 4 u (|w xh| + |b|), then h(T) |y|.
* dx = s (a - xh c1 - c2):  a, c1, c2 by the same sums; dgain, dbias: chains of at most 200 + rows / 64
  additions (64 or more partial sums per column for long inputs).
Second-order terms are covered by a factor 1.1.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
# a row in one lane, odd and even, each number of elements a lane, borders of one wavefront and of a workgroup
DIMS = [1, 2, 7, 8, 64, 100, 513, 1001, 1024, 2047, 2048, 2056, 2560, 4099, 8192, 8200]
TINY = {torch.float32: 1e-38, torch.bfloat16: 1e-38, torch.float16: 2.0**-25}


def half(dtype):
    return torch.finfo(dtype).eps / 2


def make(shape, dtype, seed, per_group, bias=True, wdtype=None):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(shape, generator=g) * torch.exp(torch.randn(*shape[:-1], 1, generator=g)) + 0.5).to(dtype)
    pshape = (shape[0], shape[-1]) if per_group else (shape[-1],)
    w = (1.0 + 0.3 * torch.randn(pshape, generator=g)).to(wdtype or dtype)
    b = (0.2 * torch.randn(pshape, generator=g)).to(wdtype or dtype) if bias else None
    dy = torch.randn(shape, generator=g).to(dtype)
    return x, w, b, dy


def reference(x, w, b, dy, eps, rms, offset):
    """Values and bounds in 64 bits: {name: (value, bound)} for y, dx, dw, db."""
    X, DY = x.double(), dy.double()
    D = X.shape[-1]
    per_group = w is not None and w.dim() == 2 or b is not None and b.dim() == 2

    def rows_of(p, fill):
        if p is None:
            return torch.full((D,), fill, dtype=torch.float64)
        p = p.double()
        return p.reshape(p.shape[0], *([1] * (X.dim() - 2)), D) if per_group else p

    W = rows_of(w, 1.0) + (offset if w is not None else 0.0)
    B = rows_of(b, 0.0)
    mu = torch.zeros_like(X[..., :1]) if rms else X.mean(-1, keepdim=True)
    s = 1.0 / torch.sqrt(((X - mu) ** 2).mean(-1, keepdim=True) + eps)
    xh = (X - mu) * s
    dmu = 0.0 if rms else 57 * U * X.abs().mean(-1, keepdim=True) * s
    e = dmu + xh.abs() * (dmu + 40 * U)
    y = xh * W + B
    T = half(x.dtype)
    tiny = TINY[x.dtype]
    out = {"y": (y, 1.1 * (W.abs() * e + 4 * U * ((W * xh).abs() + B.abs())) + T * y.abs() * 1.01 + tiny)}
    a = DY * W
    c1 = (a * xh).mean(-1, keepdim=True)
    c2 = torch.zeros_like(c1) if rms else a.mean(-1, keepdim=True)
    dx = s * (a - xh * c1 - c2)
    dc1 = 60 * U * (a * xh).abs().mean(-1, keepdim=True) + (a.abs() * e).mean(-1, keepdim=True)
    dc2 = 0.0 if rms else 60 * U * a.abs().mean(-1, keepdim=True)
    terms = a.abs() + (xh * c1).abs() + c2.abs()
    bound = s * (3 * U * a.abs() + e * c1.abs() + xh.abs() * dc1 + dc2 + 6 * U * terms) + (dmu + 40 * U) * dx.abs()
    out["dx"] = (dx, 1.1 * bound + T * dx.abs() * 1.01 + tiny)
    red = tuple(range(1, X.dim() - 1)) if per_group else tuple(range(X.dim() - 1))
    rows = 1
    for i in red:
        rows *= X.shape[i]
    chain = (200 + rows / 64) * U
    for name, p, t, extra in (("dw", w, DY * xh, DY.abs() * e), ("db", b, DY, torch.zeros_like(DY))):
        if p is not None:
            v = t.sum(red) if red else t
            bound = (chain * t.abs().sum(red) + extra.sum(red)) if red else chain * t.abs() + extra
            out[name] = (v, 1.1 * bound + half(p.dtype) * v.abs() * 1.01 + TINY[p.dtype])
    return out


def check(got, want, what):
    value, bound = want
    got = got.detach().double().cpu()
    assert got.shape == value.shape, what
    over = (got - value).abs() / bound
    assert bool((over <= 1).all()), f"{what}: {float(over.max()):.3g} times the bound"


def run(x, w, b, dy, eps, kind, dev):
    from unirl_amd import models

    leaves = [t.to(dev).requires_grad_(True) if t is not None else None for t in (x, w, b)]
    X, W, B = leaves
    if kind == "rms":
        y = models.rms_norm(X, W, eps)
    elif kind == "rms1":
        y = models.rms_norm(X, W, eps, unit_offset=True)
    elif kind == "mod":
        y = models.modulated_layer_norm(X, W, B, eps)
    else:
        y = models.layer_norm(X, W, B, eps)
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy.to(dev))
    names = [n for n, t in zip(("dx", "dw", "db"), leaves) if t is not None]
    return {"y": y, **dict(zip(names, grads))}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", DIMS)
@pytest.mark.parametrize("kind", ["layer", "rms", "mod"])
def test_values_and_gradients(dev, kind, D, dtype):
    shape = (3, 5, D) if kind == "mod" else (13, D)
    x, w, b, dy = make(shape, dtype, D, kind == "mod", bias=kind != "rms")
    eps = 1e-5
    want = reference(x, w, b, dy, eps, kind == "rms", 1.0 if kind == "mod" else 0.0)
    got = run(x, w, b, dy, eps, kind, dev)
    for name in want:
        check(got[name], want[name], f"{kind} {D} {dtype} {name}")
    assert got["y"].dtype == dtype and got["dx"].dtype == dtype and got["dw"].dtype == w.dtype


@pytest.mark.parametrize("D", [16384, 16392, 32768])
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_longest_rows(dev, kind, D):
    for dtype in DTYPES:
        x, w, b, dy = make((3, D), dtype, D, False, bias=kind != "rms")
        want = reference(x, w, b, dy, 1e-5, kind == "rms", 0.0)
        got = run(x, w, b, dy, 1e-5, kind, dev)
        for name in want:
            check(got[name], want[name], f"{kind} {D} {dtype} {name}")


@pytest.mark.parametrize("kind", ["layer", "rms", "mod"])
@pytest.mark.parametrize("D", [10240, 10241, 12296, 16383, 16385, 24576, 24579, 32760, 32767])
def test_long_rows_several_a_workgroup(dev, D, kind):
    """More rows than workgroups of one row each stay resident: every one takes two or three in turn."""
    for dtype in (torch.float32, torch.bfloat16):
        x, w, b, dy = make((2, 300, D) if kind == "mod" else (520, D), dtype, D, kind == "mod", bias=kind != "rms")
        want = reference(x, w, b, dy, 1e-5, kind == "rms", 1.0 if kind == "mod" else 0.0)
        got = run(x, w, b, dy, 1e-5, kind, dev)
        for name in want:
            check(got[name], want[name], f"{kind} {D} {dtype} {name}")


def test_longer_rows_are_refused(dev):
    from unirl_amd import models

    with pytest.raises(ValueError, match="limit"):
        models.layer_norm(torch.ones(2, 32769, device=dev))


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 63, 1025, 20011])
@pytest.mark.parametrize("D", [40, 2560])
def test_numbers_of_rows(dev, rows, D):
    x, w, b, dy = make((rows, D), torch.bfloat16, rows, False)
    want = reference(x, w, b, dy, 1e-6, False, 0.0)
    got = run(x, w, b, dy, 1e-6, "layer", dev)
    for name in want:
        check(got[name], want[name], f"{rows} {D} {name}")


@pytest.mark.parametrize("wdtype", DTYPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_parameters_of_another_type_and_missing_ones(dev, dtype, wdtype):
    x, w, b, dy = make((9, 264), dtype, 3, False, wdtype=wdtype)
    for ww, bb in ((w, b), (w, None), (None, b), (None, None)):
        want = reference(x, ww, bb, dy, 1e-5, False, 0.0)
        got = run(x, ww, bb, dy, 1e-5, "layer", dev)
        for name in want:
            check(got[name], want[name], f"{dtype} {wdtype} {name}")
    want = reference(x, w, None, dy, 1e-5, True, 1.0)
    got = run(x, w, None, dy, 1e-5, "rms1", dev)
    for name in want:
        check(got[name], want[name], f"1 + weight {name}")


def test_strided_views_are_read_in_place(dev):
    """Slices over rows and columns, swapped dimensions, a broadcast gradient, halves of one projection."""
    from unirl_amd import models, ops

    g = torch.Generator().manual_seed(5)
    big = torch.randn(4, 9, 72, generator=g).bfloat16().to(dev)
    w = torch.randn(64, generator=g).bfloat16().to(dev)
    views = {
        "rows": big[:, 2:7, :64], "odd columns": big[:, 1:, 3:67], "swapped": big[..., :64].transpose(0, 1),
        "one row": big[:, 4, :64], "step": big[:, ::2, :64], "broadcast": big[:1, :, :64].expand(4, 9, 64),
        "columns apart": big[:, :, ::2][..., :32],
    }
    for name, v in views.items():
        ww = w[: v.shape[-1]]
        y, mean, rstd = ops.layer_norm(v, ww, None, want_stats=True)
        c = v.contiguous()
        y2, mean2, rstd2 = ops.layer_norm(c, ww, None, want_stats=True)
        assert torch.equal(mean, mean2) and torch.equal(rstd, rstd2) or name == "odd columns", name
        want = reference(c.cpu(), ww.cpu(), None, c.cpu(), 1e-5, False, 0.0)
        check(y, want["y"], name)
        one = torch.ones((), device=dev, dtype=v.dtype).expand(v.shape)
        dx, dw, _ = ops.layer_norm_bwd(one, v, mean, rstd, ww)
        want = reference(c.cpu(), ww.cpu(), None, one.cpu(), 1e-5, False, 0.0)
        check(dx, want["dx"], name)
        check(dw, want["dw"], name)
        # dy strided unlike x
        dy = torch.randn(v.shape[::-1], generator=g).bfloat16().to(dev).permute(*range(v.dim() - 1, -1, -1))
        dx, dw, _ = ops.layer_norm_bwd(dy, v, mean, rstd, ww)
        want = reference(c.cpu(), ww.cpu(), None, dy.cpu(), 1e-5, False, 0.0)
        check(dx, want["dx"], name)
        check(dw, want["dw"], name)
    both = torch.randn(4, 128, generator=g).bfloat16().to(dev)
    scale, shift = both.chunk(2, dim=1)
    x = big[:, :, :64]
    y = models.modulated_layer_norm(x, scale, shift)
    want = reference(x.cpu(), scale.cpu(), shift.cpu(), x.cpu(), 1e-6, False, 1.0)
    check(y, want["y"], "halves of one projection")
    assert torch.equal(y, models.modulated_layer_norm(x, scale[:, None], shift[:, None]))


def test_many_groups(dev):
    """More groups than one launch takes, and groups of one row."""
    x, w, b, dy = make((70001, 1, 8), torch.float32, 2, True)
    want = reference(x, w, b, dy, 1e-5, False, 1.0)
    from unirl_amd import models, ops

    y = models.modulated_layer_norm(x.to(dev), w.to(dev), b.to(dev), 1e-5)
    check(y, want["y"], "y")
    _, mean, rstd = ops.layer_norm(x.to(dev), w.to(dev), b.to(dev), eps=1e-5, unit_offset=True, want_stats=True)
    with pytest.raises(ValueError, match="limit"):
        ops.layer_norm_bwd(dy.to(dev), x.to(dev), mean, rstd, w.to(dev), b.to(dev), unit_offset=True)
    dx, _, _ = ops.layer_norm_bwd(dy[:65535].to(dev), x[:65535].to(dev), mean[:65535], rstd[:65535], w[:65535].to(dev),
                                  b[:65535].to(dev), unit_offset=True)
    check(dx, tuple(t[:65535] for t in want["dx"]), "dx")


def test_empty_inputs(dev):
    from unirl_amd import models

    w, b = torch.ones(8, device=dev, requires_grad=True), torch.zeros(8, device=dev, requires_grad=True)
    x = torch.empty(0, 8, device=dev, requires_grad=True)
    y = models.layer_norm(x, w, b)
    assert y.shape == (0, 8)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty(0, 8, device=dev))
    assert dx.shape == (0, 8) and not dw.any() and not db.any()
    s = torch.zeros(2, 8, device=dev, requires_grad=True)
    y = models.modulated_layer_norm(torch.empty(2, 0, 8, device=dev), s, torch.zeros(2, 8, device=dev))
    (ds,) = torch.autograd.grad(y, s, torch.empty(2, 0, 8, device=dev))
    assert y.shape == (2, 0, 8) and ds.shape == (2, 8) and not ds.any()
    with pytest.raises(ValueError):
        models.layer_norm(torch.empty(3, 0, device=dev))


def test_constant_rows_large_values_and_bad_ones(dev):
    """A row without variance gives the bias; an infinity or NaN stays in its row and in the gradients
    that read it; an offset a thousand times the spread costs no more than its bound says."""
    from unirl_amd import models

    x = torch.randn(6, 264)
    x[1] = 3.0
    x[2, 7] = float("inf")
    x[3, 0] = float("nan")
    x[4] += 1000.0
    x[5] = 0.0
    w, b = torch.rand(264) + 0.5, torch.randn(264)
    y = models.layer_norm(x.to(dev), w.to(dev), b.to(dev)).cpu()
    assert torch.equal(y[1], b) and torch.equal(y[5], b)
    assert torch.isnan(y[2]).all() and torch.isnan(y[3]).all()
    want = reference(x[[0, 4]], w, b, torch.zeros(2, 264), 1e-5, False, 0.0)
    check(y[[0, 4]], want["y"], "offset")
    # RMS norm of an infinite element: x / inf is 0 elsewhere, NaN there, as the formula says
    y = models.rms_norm(x.to(dev), w.to(dev)).cpu()
    assert torch.isnan(y[2, 7]) and not y[2, :7].any() and torch.isnan(y[3]).all() and not y[5].any()


@pytest.mark.parametrize("dtype,D", [(torch.float32, 256), (torch.float32, 8), (torch.float32, 2048), (torch.float32, 8192),
                                     (torch.bfloat16, 32), (torch.bfloat16, 256), (torch.bfloat16, 1024), (torch.float32, 1)])
def test_gradient_of_large_constant_rows(dev, dtype, D):
    """Rows of 2^123: the mean is exact (D is a power of two), the variance 0 and rstd 1 / sqrt(eps); lanes behind
    the row's end must not bring in (0 - mean) rstd, which overflows.  dx = (a - mean(a)) / sqrt(eps)."""
    x = torch.full((5, D), 2.0**123).to(dtype)
    _, w, b, dy = make((5, D), dtype, D, False)
    got = run(x, w, b, dy, 2.0**-18, "layer", dev)
    a = dy.double() * w.double()
    want = (a - a.mean(-1, keepdim=True)) * 2.0**9
    # products and sums of a as in the module's comment, scaled by rstd; the value rounded to dtype
    bound = 512 * U * (6 * a.abs() + 60 * a.abs().mean(-1, keepdim=True)) + half(dtype) * want.abs() * 1.01 + 1e-30
    check(got["dx"], (want, bound), "dx")
    assert not got["dw"].any()
    check(got["db"], (dy.double().sum(0), 8 * U * dy.double().abs().sum(0) + half(dtype) * dy.double().sum(0).abs() * 1.01 + 1e-30),
          "db")


def test_gradient_against_differences(dev):
    """<dx, d> from the kernel against (f(x + t d) - f(x - t d)) / 2t of the 64-bit formula, t = 2^-20: the
    difference's own error is t^2 times the third derivative (below 1e-9 here) plus 2^-52 |f| / t."""
    x, w, b, dy = make((7, 120), torch.float32, 11, False)
    got = run(x, w, b, dy, 1e-5, "layer", dev)
    want = reference(x, w, b, dy, 1e-5, False, 0.0)
    g = torch.Generator().manual_seed(12)
    t = 2.0**-20

    def f(xx, ww, bb):
        d = xx - xx.mean(-1, keepdim=True)
        yy = d / torch.sqrt((d * d).mean(-1, keepdim=True) + 1e-5) * ww + bb
        return (yy * dy.double()).sum()

    args = [x.double(), w.double(), b.double()]
    for i, name in enumerate(("dx", "dw", "db")):
        d = torch.randn(args[i].shape, generator=g).double()
        up, dn = list(args), list(args)
        up[i], dn[i] = args[i] + t * d, args[i] - t * d
        diff = float((f(*up) - f(*dn)) / (2 * t))
        mine = float((got[name].double().cpu() * d).sum())
        bound = float((want[name][1] * d.abs()).sum()) + 1e-6 * (1.0 + abs(diff))
        assert abs(mine - diff) <= bound, (name, mine, diff, bound)


def test_same_bits_every_time_and_on_another_stream(dev):
    x, w, b, dy = make((5000, 1001), torch.bfloat16, 4, False)
    first = run(x, w, b, dy, 1e-5, "layer", dev)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        second = run(x, w, b, dy, 1e-5, "layer", dev)
    torch.cuda.synchronize()
    for name in first:
        assert torch.equal(first[name], second[name]), name


def test_captured_forward_and_backward(dev):
    """Two graphs of the same shapes, replayed in turn with eager calls between, against eager results."""
    from unirl_amd import ops

    x = torch.empty(600, 520, device=dev, dtype=torch.bfloat16)
    dy, w = torch.empty_like(x), torch.rand(520, device=dev).bfloat16()

    def step():
        y, mean, rstd = ops.layer_norm(x, w, None, rms=True, want_stats=True)
        return (y, *ops.layer_norm_bwd(dy, x, mean, rstd, w, rms=True)[:2])

    def fill(seed):
        g = torch.Generator().manual_seed(seed)
        x.copy_(torch.randn(x.shape, generator=g))
        dy.copy_(torch.randn(x.shape, generator=g))

    fill(0)
    step()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for seed in range(1, 5):
        fill(seed)
        for graph, out in graphs:
            for o in out:
                o.zero_()
            graph.replay()
            torch.cuda.synchronize()
            for o, e in zip(out, step()):
                assert torch.equal(o, e)


def test_captured_autograd_and_a_living_eager_graph(dev):
    """A captured backward is refused while a graph of the default stream over the same leaf is alive;
    without one it is captured, and every replay gives the eager gradients."""
    from unirl_amd import models

    x = torch.randn(300, 520, device=dev).bfloat16()
    dy = torch.randn_like(x)
    w = torch.rand(520, device=dev).bfloat16().requires_grad_(True)

    alive = models.rms_norm(x, w)
    refused = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(refused):
        y = models.rms_norm(x, w)
        with pytest.raises(RuntimeError, match="alive"):
            y.backward(dy)
    assert w.grad is None
    del alive, y, refused

    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        models.rms_norm(x, w).backward(dy)
    held = w.grad
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        x.copy_(torch.randn(x.shape, generator=g))
        dy.copy_(torch.randn(x.shape, generator=g))
        held.zero_()
        graph.replay()
        torch.cuda.synchronize()
        want = torch.autograd.grad(models.rms_norm(x, w), w, dy)[0]
        assert torch.equal(held, want)


@pytest.mark.parametrize("bias", [False, True])
def test_backward_stays_inside_its_scratch(dev, bias):
    """Scratch of exactly the documented size: the bytes behind it keep their values (and the entry point
    itself refuses a launch whose partial rows would not fit)."""
    import ctypes

    from unirl_amd import _native as N
    from unirl_amd import ops

    for dtype in (torch.bfloat16, torch.float32):
        for D in (8, 64, 100, 264, 513, 1024, 1536, 2048, 2304, 2560, 2568, 2600, 3200, 3333, 4096, 4608, 5120, 7168, 8192, 10240):
            for G, R in ((1, 3000), (3, 1100)):
                x = torch.randn(G * R, D, device=dev).to(dtype)
                w = torch.ones(D, device=dev, dtype=dtype)
                _, mean, rstd = ops.layer_norm(x, w, w, want_stats=True)
                size = int(N.lib().unirl_layer_norm_bwd_scratch_bytes(G, R, D))
                scratch = torch.full((size + 4096,), 77, dtype=torch.uint8, device=dev)
                dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
                desc = N.NormDesc(x=N.ptr(x), dtype=N.dtype_code(dtype), x_group_stride=R * D, x_row_stride=D, groups=G, rows=R, D=D,
                                  gain=N.ptr(w), gain_dtype=N.dtype_code(dtype), center=1, mean=N.ptr(mean), rstd=N.ptr(rstd))
                rc = N.lib().unirl_layer_norm_bwd(ctypes.byref(desc), N.ptr(x), R * D, D, N.ptr(dx), N.ptr(dw),
                                                  N.ptr(db) if bias else None, 0, N.ptr(scratch), size, N.current_stream(dev))
                assert rc == 0, (D, G, R, rc)
                assert bool((scratch[size:] == 77).all()), (D, G, R)


def test_rows_outside_a_view_stay_untouched_and_refusals(dev):
    from unirl_amd import models, ops

    x = torch.randn(4, 16, device=dev)
    for bad in (
        lambda: models.layer_norm(x, torch.ones(15, device=dev)),
        lambda: ops.layer_norm(x, torch.ones(3, 16, device=dev)),
        lambda: ops.layer_norm(x, torch.ones(16, device=dev), torch.ones(16, device=dev).bfloat16()),
        lambda: ops.layer_norm(x, torch.ones(16, device=dev), torch.ones(4, 16, device=dev)),
        lambda: ops.layer_norm_bwd(x[:2], x, None, torch.ones(4, device=dev), rms=True),
        lambda: ops.layer_norm_bwd(x, x, None, torch.ones(4, device=dev)),
        lambda: ops.layer_norm_bwd(x, x, torch.ones(3, device=dev), torch.ones(4, device=dev)),
    ):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        models.layer_norm(x.double())
    with pytest.raises(TypeError):
        models.layer_norm(x, torch.ones(16, device=dev).double())
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        models.layer_norm(x, torch.ones(16))
    # a second derivative is not offered
    x.requires_grad_(True)
    (gx,) = torch.autograd.grad(models.layer_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gx.sum(), x)


def test_autograd_asks_for_what_it_needs(dev):
    """Every choice of inputs that want a gradient, twice through one graph; an input written between
    forward and backward is noticed; checkpointing recomputes the node."""
    from torch.utils.checkpoint import checkpoint

    from unirl_amd import models

    x, w, b, dy = make((33, 136), torch.bfloat16, 21, False)
    want = reference(x, w, b, dy, 1e-5, False, 0.0)
    for mask in range(1, 8):
        leaves = [t.to(dev).requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, w, b))]
        y = models.layer_norm(*leaves)
        asked = [(n, t) for n, t in zip(("dx", "dw", "db"), leaves) if t.requires_grad]
        for keep in (True, False):
            grads = torch.autograd.grad(y, [t for _, t in asked], dy.to(dev), retain_graph=keep)
            for (name, _), g in zip(asked, grads):
                check(g, want[name], f"{name} of mask {mask}")
        with torch.no_grad():
            assert not models.layer_norm(*leaves).requires_grad
    for i in range(2):  # x and the gain are read again by the backward
        leaves = [t.to(dev).requires_grad_(True) for t in (x, w, b)]
        y = models.layer_norm(*leaves)
        with torch.no_grad():
            leaves[i].add_(1.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward(dy.to(dev))
    leaves = [t.to(dev).requires_grad_(True) for t in (x, w, b)]
    y = checkpoint(models.layer_norm, *leaves, use_reentrant=False)
    for name, g in zip(("dx", "dw", "db"), torch.autograd.grad(y, leaves, dy.to(dev))):
        check(g, want[name], f"checkpointed {name}")


def test_rms_norm_with_a_bias_and_modulation_in_other_shapes(dev):
    from unirl_amd import models, ops

    x, w, b, dy = make((19, 200), torch.float16, 22, False)
    want = reference(x, w, b, dy, 1e-5, True, 0.0)
    args = [t.to(dev) for t in (x, w, b)]
    y, mean, rstd = ops.layer_norm(*args, rms=True, want_stats=True)
    assert mean is None
    check(y, want["y"], "y")
    got = ops.layer_norm_bwd(dy.to(dev), args[0], None, rstd, *args[1:], rms=True)
    for name, g in zip(("dx", "dw", "db"), got):
        check(g, want[name], name)
    # [B, D], [B, h, w, D], a permuted [B, D, h, w] and a gain broadcast over the samples
    for shape in ((5, 72), (3, 2, 5, 72)):
        x, w, b, dy = make(shape, torch.bfloat16, 23, True)
        want = reference(x, w, b, dy, 1e-6, False, 1.0)
        got = run(x, w, b, dy, 1e-6, "mod", dev)
        for name in want:
            check(got[name], want[name], f"{shape} {name}")
    picture = x.permute(0, 3, 1, 2).contiguous().to(dev).permute(0, 2, 3, 1)
    assert not picture.is_contiguous()
    check(models.modulated_layer_norm(picture, w.to(dev), b.to(dev)), want["y"], "permuted")
    one_w, one_b = w[:1].to(dev).requires_grad_(True), b[:1].to(dev).requires_grad_(True)
    y = models.modulated_layer_norm(x.to(dev), one_w.expand(3, 72), one_b.expand(3, 72))
    gw, gb = torch.autograd.grad(y, (one_w, one_b), dy.to(dev))
    same = reference(x, w[:1].expand(3, 72), b[:1].expand(3, 72), dy, 1e-6, False, 1.0)
    check(y, same["y"], "one modulation")
    for g, name in ((gw, "dw"), (gb, "db")):  # the sum over samples is autograd's, in bf16: one rounding more per sample
        value, bound = same[name]
        check(g, (value.sum(0, keepdim=True), bound.sum(0, keepdim=True) + 3 * half(torch.bfloat16) * value.abs().sum(0, keepdim=True)),
              name)


def test_replay_log_prob_behind_a_final_norm(dev):
    """chunked_replay_logp(final_norm=...) on hidden states from before the norm: the same log-probs and
    gradients as the norm called in front of it, and the gain's gradient."""
    from unirl_amd import models
    from unirl_amd.models.ar_logp import _apply_final_norm

    g = torch.Generator().manual_seed(9)
    hidden = torch.randn(2, 21, 128, generator=g).bfloat16().to(dev)
    tokens = torch.randint(0, 997, (2, 20), generator=g).to(dev)
    head = torch.nn.Linear(128, 997, bias=False, device=dev, dtype=torch.bfloat16)
    for norm in (torch.nn.RMSNorm(128, eps=1e-6), torch.nn.RMSNorm(128), torch.nn.LayerNorm(128),
                 torch.nn.LayerNorm(128, elementwise_affine=False)):
        norm = norm.to(dev, torch.bfloat16)
        h = hidden.clone().requires_grad_(True)
        out = models.chunked_replay_logp(head, h, tokens, 0.9, final_norm=norm)
        leaves = [h, head.weight, *norm.parameters()]
        got = torch.autograd.grad(out.sum(), leaves)
        if isinstance(norm, torch.nn.LayerNorm):
            y = models.layer_norm(h[:, :20], norm.weight, norm.bias, norm.eps)
        else:
            y = models.rms_norm(h[:, :20], norm.weight, norm.eps or torch.finfo(torch.float32).eps)
        plain = models.chunked_replay_logp(head, y, tokens, 0.9)
        assert torch.equal(out, plain)
        for a, b in zip(got, torch.autograd.grad(plain.sum(), leaves)):
            assert torch.equal(a, b)
        assert not got[0][:, 20:].any()
        with torch.no_grad():
            scored = models.chunked_replay_logp(head, h, tokens, 0.9, final_norm=norm)
            assert torch.equal(scored, models.chunked_replay_logp(head, y.detach(), tokens, 0.9))
    # small states, where the module's default eps counts: two roundings to bf16 apart from the module at most
    small = (torch.randn(2, 20, 128, generator=g) * 2e-3).bfloat16().to(dev)
    for norm in (torch.nn.RMSNorm(128), torch.nn.LayerNorm(128)):
        norm = norm.to(dev, torch.bfloat16)
        got = _apply_final_norm(norm, small).float()
        assert bool(((got - norm(small).float()).abs() <= 2 * 2.0**-8 * 1.01 * got.abs() + 1e-6).all())
    called = []

    def other(t):
        called.append(tuple(t.shape))
        return t * 2

    out = models.chunked_replay_logp(head, hidden, tokens, final_norm=other)
    assert called == [(2, 20, 128)]
    assert torch.equal(out, models.chunked_replay_logp(head, hidden[:, :20] * 2, tokens))

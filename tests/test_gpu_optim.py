"""The gradients' global norm and the AdamW step (32- and 8-bit moments) against 64-bit formulas.

Tolerances, u = 2^-24, h(T) = finfo(T).eps / 2.  The clip factor c carries at most 5 u (norm, sum, quotient and
the product with g), so g' = c g is off by 5 u relative (0 without clipping; 5 u is allowed throughout).
  m = b1 m + (1 - b1) g':  constants, products and sum round once each: 9 u (|b1 m| + |(1 - b1) g'|) =: em
  v = b2 v + (1 - b2) g'^2: 15 u v
  p: 3 u |p| + step ((em + 16 u |m|) / denom), then h(T) |p| where p is held in 16 bits
with denom's relative error 7.5 u (root of v) + 4 u included in the 16 u.  Second order: factor 1.05.

8-bit moments: with x the exact new moment over the block's scale, s its code step and w the 16 dither bits,
the code is floor(x / s + w / 2^16).  x / s < 16 carries 15 u relative and the lower 4 bits of x are cut:
the code may differ from the exact one only where x / s + w / 2^16 lies within
16 * 15 * 2^-24 + 2^-20 + 2^-20 < 2^-15 of an integer, and then by one step; a scale only where the block's largest
value lies within 15 u of a power of two.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
BLOCK = 256
SIZES = [1, 3, 4, 255, 256, 257, 1023, 1024, 4096, 4097, 10007]
TINY = {torch.float32: 1e-38, torch.bfloat16: 1e-38, torch.float16: 2.0**-25}


def half(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------ restatement of the formats (CPU, 64 bits)
def mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & 0xFFFFFFFF
    return x ^ (x >> 16)


def dither(n, base, seed, step):
    """(w for m, w for v) as 16-bit integers, for elements [0, n) of a tensor whose index base is `base`."""
    key = mix(torch.tensor((seed + step * 0x9E3779B9) & 0xFFFFFFFF))
    i = torch.arange(n, dtype=torch.int64) + base
    key = (key + (i >> 32) * 0x9E3779B9) & 0xFFFFFFFF
    h = mix((i & 0xFFFFFFFF) ^ key)
    return h & 0xFFFF, h >> 16


def decode(code, scale, which):
    code, n = code.reshape(-1).long().cpu(), code.numel()
    ebits = 4 if which == "m" else 5
    e, f = (code >> 3) % 2**ebits, (code & 7).double()
    bias = 2 ** (ebits - 1) - 1
    v = torch.where(e > 0, (8 + f), f) * torch.pow(2.0, (e.clamp(min=1) - bias - 3).double())
    if which == "m":
        v = torch.where(code >= 128, -v, v)
        v[(code & 127) == 127] = math.nan
    else:
        v[code == 0xF8] = math.inf
        v[code > 0xF8] = math.nan
    return v * torch.pow(2.0, scale.cpu().double() - 127).repeat_interleave(BLOCK)[:n]


def expected_codes(x, w, which):
    """(values, step of each, distance of x / s + w / 2^16 from an integer, scale bytes, doubtful blocks)."""
    n, top, low = x.numel(), (7 if which == "m" else 14), (-6 if which == "m" else -14)
    pad = torch.zeros(-(-n // BLOCK) * BLOCK, dtype=torch.float64)
    pad[:n] = x.abs()
    most = pad.view(-1, BLOCK).amax(1)
    mant, e = torch.frexp(most)
    k = torch.where(most > 0, (e - 1 - top).clamp(min=-126), torch.full_like(e, -126))
    doubtful = (mant > 1 - 16 * U) | (mant < 0.5 * (1 + 16 * U))
    unit = torch.pow(2.0, k.double()).repeat_interleave(BLOCK)[:n]
    a = x.abs() / unit
    _, ea = torch.frexp(a)
    s = torch.pow(2.0, (ea - 1).clamp(min=low).double() - 3)
    q = a / s + w.double() / 65536
    value = torch.floor(q) * s
    if which == "v":
        value = torch.where(x > 0, value.clamp(min=2.0**-17), value)
    return torch.sign(x) * value * unit, s * unit, (q - q.round()).abs(), (k + 127).to(torch.uint8), doubtful


def make(sizes, dtype, gdtype, bits, master, seed, dev, misalign=False):
    g = torch.Generator().manual_seed(seed)
    T = []
    for i, n in enumerate(sizes):
        sc = math.exp(float(torch.randn((), generator=g)) - 5)
        t = {"grad": (torch.randn(n, generator=g) * sc).to(gdtype)}
        p = torch.randn(n, generator=g) * 0.05
        t["param"] = p.to(dtype)
        if master:
            t["master"] = p
        m, v = torch.randn(n, generator=g) * 0.3 * sc, (torch.randn(n, generator=g) ** 2 + 0.05) * sc * sc
        if bits == 32:
            t["m"], t["v"] = m, v
        else:
            blocks = -(-n // BLOCK)
            t["m"] = torch.randint(0, 256, (n,), generator=g, dtype=torch.uint8)
            t["m"][(t["m"] & 127) == 127] = 3  # no NaN
            t["v"] = torch.randint(0, 0xF1, (n,), generator=g, dtype=torch.uint8)
            t["ms"] = torch.randint(100, 112, (blocks,), generator=g, dtype=torch.uint8)
            t["vs"] = torch.randint(80, 95, (blocks,), generator=g, dtype=torch.uint8)
        T.append(t)

    def place(t):
        if not misalign:
            return t.to(dev)
        buf = torch.zeros(t.numel() + 1, dtype=t.dtype, device=dev)
        buf[1:] = t.to(dev)
        return buf[1:]

    return T, [{k: place(v) for k, v in t.items()} for t in T]


def reference(t, hyper, c, base):
    """What the step makes of one tensor: {name: (value, bound)}, and the exact new moments."""
    lr, (b1, b2), eps, wd, step = (hyper[k] for k in ("lr", "betas", "eps", "weight_decay", "step"))
    g = t["grad"].double() * c
    m = t["m"].double() if "ms" not in t else decode(t["m"], t["ms"], "m")
    v = t["v"].double() if "ms" not in t else decode(t["v"], t["vs"], "v")
    p = (t["master"] if "master" in t else t["param"]).double()
    em = 9 * U * ((b1 * m).abs() + ((1 - b1) * g).abs())
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    denom = torch.sqrt(v) / math.sqrt(1 - b2**step) + eps
    size = lr / (1 - b1**step)
    new = p * (1 - lr * wd) - size * m / denom
    bound = 3 * U * p.abs() + size * (em + 16 * U * m.abs()) / denom + U * new.abs()
    out = {"param": (new, 1.05 * bound + half(t["param"].dtype) * new.abs() * 1.01 + TINY[t["param"].dtype])}
    if "master" in t:
        out["master"] = (new, 1.05 * bound)
    if "ms" not in t:
        out["m"], out["v"] = (m, 1.05 * em + 1e-38), (v, 1.05 * 15 * U * v + 1e-38)
    return out, m, v


def check(got, want, what):
    value, bound = want
    over = (got.double().cpu() - value).abs() / bound
    assert bool((over <= 1).all()), f"{what}: {float(over.max()):.3g} times the bound"


def check_codes(code, scale, x, w, which, what):
    value, s, near, scales, doubtful = expected_codes(x, w, which)
    sure = ~doubtful
    assert torch.equal(scale.cpu()[sure], scales[sure]), what
    got = decode(code, scale, which)
    ok = sure.repeat_interleave(BLOCK)[: x.numel()]
    off = (got - value).abs()
    assert bool((off[ok] <= 1.001 * s[ok]).all()), what
    assert bool(((off == 0) | (near < 2.0**-15))[ok].all()), what
    assert float(ok.double().mean()) > 0.9 or x.numel() < 10 * BLOCK


def apply(D, hyper, **kw):
    from unirl_amd import ops

    eight = "ms" in D[0]
    ops.adamw_step(
        [t["param"] for t in D], [t["grad"] for t in D], [t["m"] for t in D], [t["v"] for t in D],
        masters=[t["master"] for t in D] if "master" in D[0] else None,
        exp_avg_scales=[t["ms"] for t in D] if eight else None, exp_avg_sq_scales=[t["vs"] for t in D] if eight else None,
        **hyper, **kw)


HYPER = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1, step=3)
KINDS = [(torch.float32, torch.float32, False)] + [
    (d, g, master) for d in (torch.bfloat16, torch.float16) for g in (d, torch.float32) for master in (False, True)]


@pytest.mark.parametrize("misalign", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,gdtype,master", KINDS)
def test_step(dev, dtype, gdtype, master, bits, misalign):
    T, D = make(SIZES, dtype, gdtype, bits, master, 7, dev, misalign)
    apply(D, HYPER, seed=99)
    base = 0
    for i, (t, d) in enumerate(zip(T, D)):
        want, m, v = reference(t, HYPER, 1.0, base)
        for name in want:
            check(d[name], want[name], f"{name} of tensor {i}")
        if bits == 8:
            wm, wv = dither(m.numel(), base, 99, HYPER["step"])
            check_codes(d["m"], d["ms"], m, wm, "m", f"m of tensor {i}")
            check_codes(d["v"], d["vs"], v, wv, "v", f"v of tensor {i}")
        base += -(-m.numel() // BLOCK) * BLOCK


def test_neighbours_stay_untouched(dev):
    """What lies before and behind each tensor in its buffer keeps its bytes."""
    for bits in (32, 8):
        T, D = make([5, 257, 1021], torch.bfloat16, torch.bfloat16, bits, True, 3, dev)
        guards = []
        for d in D:
            for k in list(d):
                if k == "grad":
                    continue
                buf = torch.full((d[k].numel() + 32,), 77, dtype=d[k].dtype, device=dev)
                buf[16:-16] = d[k]
                d[k] = buf[16:-16]
                guards.append(buf)
        apply(D, HYPER)
        torch.cuda.synchronize()
        for buf in guards:
            assert bool((buf[:16] == 77).all()) and bool((buf[-16:] == 77).all())


@pytest.mark.parametrize("count", [1, 47, 48, 49, 160, 161, 400])
def test_many_tensors(dev, count):
    """More tensors than one launch takes, empty ones among them; the norm and the clipped step."""
    from unirl_amd import ops

    sizes = [(i * 131) % 700 if i % 9 else 0 for i in range(count)] if count > 1 else [5000]
    T, D = make(sizes, torch.float32, torch.float32, 32, False, count, dev)
    norm = ops.grad_norm([d["grad"] for d in D])
    exact = math.sqrt(sum(float((t["grad"].double() ** 2).sum()) for t in T))
    assert abs(float(norm) - exact) <= 1.01 * U * exact
    max_norm = 0.25 * exact
    apply(D, HYPER, grad_norm=norm, max_norm=max_norm)
    c = max_norm / (exact + 1e-6)
    for i, (t, d) in enumerate(zip(T, D)):
        want, _, _ = reference(t, HYPER, c, 0)
        for name in want:
            check(d[name], want[name], f"{name} of tensor {i}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 7, 8, 2047, 8191, 8192, 8193, 100003, 3000001])
def test_grad_norm(dev, n, dtype):
    from unirl_amd import ops

    g = torch.randn(n, generator=torch.Generator().manual_seed(n)).to(dtype)
    exact = float((g.double() ** 2).sum().sqrt())
    got = [ops.grad_norm([g.to(dev)])]
    buf = torch.zeros(n + 1, dtype=dtype, device=dev)
    buf[1:] = g.to(dev)
    got.append(ops.grad_norm([buf[1:]]))  # not aligned to the vectors
    got.append(ops.grad_norm([buf, torch.zeros(0, device=dev), torch.zeros(5, device=dev, dtype=torch.float16)]))
    for v in got:
        assert v.shape == () and v.dtype == torch.float32
        assert abs(float(v) - exact) <= 1.01 * U * exact


def test_grad_norm_of_extreme_values(dev):
    from unirl_amd import ops

    one = torch.ones(1000, device=dev)
    # squares that overflow or vanish in fp32
    assert abs(float(ops.grad_norm([one * 1e30])) / (1e30 * math.sqrt(1000)) - 1) < 2e-7
    assert abs(float(ops.grad_norm([one * 1e-30])) / (1e-30 * math.sqrt(1000)) - 1) < 2e-7
    assert float(ops.grad_norm([one * 0])) == 0.0
    assert float(ops.grad_norm([torch.zeros(0, device=dev)])) == 0.0
    bad = one.clone()
    bad[3] = float("inf")
    assert math.isinf(float(ops.grad_norm([one, bad])))
    bad[900] = float("nan")
    assert math.isnan(float(ops.grad_norm([one, bad])))
    # strides: a transposed gradient, a broadcast one
    m = torch.randn(30, 50, device=dev)
    assert float(ops.grad_norm([m.t()])) == float(ops.grad_norm([m.t().contiguous()]))
    assert float(ops.grad_norm([torch.full((), 2.0, device=dev).expand(4)])) == 4.0


def test_clip_factor(dev):
    """A norm below the bound leaves the gradient; zero, infinite and NaN norms; skipping."""
    from unirl_amd import ops

    def step(norm, max_norm=1.0, **kw):
        T, D = make([300], torch.float32, torch.float32, 32, False, 1, dev)
        apply(D, HYPER, grad_norm=torch.tensor(norm, device=dev), max_norm=max_norm, **kw)
        return T[0], D[0]

    for norm, c in ((0.5, 1.0), (0.0, 1.0), (4.0, 1.0 / (4.0 + 1e-6)), (math.inf, 0.0)):
        t, d = step(norm)
        want, _, _ = reference(t, HYPER, c, 0)
        for name in want:
            check(d[name], want[name], f"{name} at norm {norm}")
    t, d = step(math.nan)
    assert torch.isnan(d["param"]).all() and torch.isnan(d["m"]).all()
    for norm in (math.nan, math.inf):
        for max_norm in (1.0, None):
            t, d = step(norm, max_norm, skip_nonfinite=True)
            for k in ("param", "m", "v"):
                assert torch.equal(d[k].cpu(), t[k]), k
    t, d = step(2.0, None, skip_nonfinite=True)
    want, _, _ = reference(t, HYPER, 1.0, 0)
    check(d["param"], want["param"], "no bound")


def test_bad_gradients_in_8_bits(dev):
    """NaN and infinities stay with their elements: the block's other elements keep their scale."""
    T, D = make([512], torch.float32, torch.float32, 8, False, 5, dev)
    clean, C = make([512], torch.float32, torch.float32, 8, False, 5, dev)
    D[0]["grad"][10] = float("nan")
    D[0]["grad"][11] = float("inf")
    D[0]["grad"][12] = -float("inf")
    apply(D, HYPER)
    apply(C, HYPER)
    keep = torch.ones(512, dtype=torch.bool)
    keep[10:13] = False
    for k in ("m", "v", "param"):
        assert torch.equal(D[0][k].cpu()[keep], C[0][k].cpu()[keep]), k
    m, v = decode(D[0]["m"], D[0]["ms"], "m"), decode(D[0]["v"], D[0]["vs"], "v")
    assert torch.isnan(m[10:13]).all() and torch.isnan(v[10]) and torch.isinf(v[11:13]).all()


def test_blocks_of_zeros_tiny_and_huge_values(dev):
    """Zero states stay zero; blocks whose scale is at its least and large ones keep their values to a step."""
    n = 4 * BLOCK
    g = torch.zeros(n)
    g[BLOCK : 2 * BLOCK] = 1e-18  # squares below the least normal fp32 number times anything
    g[2 * BLOCK : 3 * BLOCK] = 1e15
    g[3 * BLOCK :: 2] = 1e-3
    dev_t = [dict(param=torch.zeros(n, device=dev), grad=g.to(dev), m=torch.zeros(n, dtype=torch.uint8, device=dev),
                  v=torch.zeros(n, dtype=torch.uint8, device=dev), ms=torch.zeros(4, dtype=torch.uint8, device=dev),
                  vs=torch.zeros(4, dtype=torch.uint8, device=dev))]
    hyper = dict(HYPER, step=1)
    apply(dev_t, hyper)
    d = dev_t[0]
    m, v = decode(d["m"], d["ms"], "m"), decode(d["v"], d["vs"], "v")
    wm, wv = 0.1 * g.double(), 0.001 * g.double() ** 2
    assert not m[:BLOCK].any() and not v[:BLOCK].any() and not d["param"][:BLOCK].any()
    assert not m[3 * BLOCK + 1 :: 2].any() and not v[3 * BLOCK + 1 :: 2].any()
    for part in (slice(2 * BLOCK, 3 * BLOCK), slice(3 * BLOCK, n, 2)):
        assert bool(((m - wm).abs()[part] <= wm.abs()[part] / 8).all()) and bool(((v - wv).abs()[part] <= wv[part] / 8).all())
    assert bool(((m - wm).abs()[BLOCK : 2 * BLOCK] <= wm[BLOCK : 2 * BLOCK] / 8).all())
    assert bool((v[BLOCK : 2 * BLOCK] > 0).all())  # held as the least code at least
    assert torch.isfinite(d["param"]).all()


def test_8_bit_averages_are_unbiased(dev):
    """A constant gradient for 400 steps with beta2 = 0.99: v tends to (1 - 0.99^400) g^2 = 0.982 g^2.  One
    step's rounding has a variance of at most (v / 8)^2 / 4, so the element's is at most v^2 / 256 / (1 - 0.99^2) =
    (0.443 v)^2 and that of the mean over 65536 elements (0.00173 v)^2; 6 of it are 1.1 %.  m with
    beta1 = 0.99 likewise.  (To nearest, both would stop at the first code whose step is over 1 %.)"""
    from unirl_amd import ops

    n = 65536
    g = torch.full((n,), 0.7, device=dev)
    p = torch.zeros(n, device=dev)
    st = [torch.zeros(n, dtype=torch.uint8, device=dev) for _ in range(2)]
    sc = [torch.zeros(n // BLOCK, dtype=torch.uint8, device=dev) for _ in range(2)]
    for step in range(1, 401):
        ops.adamw_step([p], [g], [st[0]], [st[1]], lr=0.0, betas=(0.99, 0.99), step=step, exp_avg_scales=[sc[0]],
                       exp_avg_sq_scales=[sc[1]], seed=5)
    m, v = ops.adamw_moments(*st, *sc)
    target = 1 - 0.99**400
    assert abs(float(m.double().mean()) / (0.7 * target) - 1) < 0.011
    assert abs(float(v.double().mean()) / (0.49 * target) - 1) < 0.011


def test_dither_depends_on_seed_step_and_position_alone(dev):
    def go(**kw):
        T, D = make([2000, 777], torch.float32, torch.float32, 8, False, 6, dev)
        apply(D, dict(HYPER, step=kw.pop("step", 3)), **kw)
        return [d["m"] for d in D], D

    a, A = go(seed=1)
    b, _ = go(seed=1)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    for kw in (dict(seed=2), dict(seed=1, step=4), dict(seed=1, index_bases=[256, 1 << 20])):
        assert not torch.equal(a[0], go(**kw)[0][0])
    # one tensor alone, with its own base, gives the same bytes as in the list; positions beyond 2^32 count
    T, D = make([2000, 777], torch.float32, torch.float32, 8, False, 6, dev)
    apply(D[1:], HYPER, seed=1, index_bases=[2048])
    assert torch.equal(D[1]["m"], a[1])
    far = go(seed=1, index_bases=[(1 << 33) + 256, 1 << 40])[1]
    for (t, d, base) in zip(T, far, [(1 << 33) + 256, 1 << 40]):
        _, m, v = reference(t, HYPER, 1.0, base)
        wm, wv = dither(m.numel(), base, 1, 3)
        check_codes(d["m"], d["ms"], m, wm, "m", "far m")
        check_codes(d["v"], d["vs"], v, wv, "v", "far v")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 255, 257, 5000])
def test_moments_every_code(dev, n, dtype):
    from unirl_amd import ops

    g = torch.Generator().manual_seed(n)
    m, v = torch.arange(n).to(torch.uint8), torch.arange(n).to(torch.uint8)
    blocks = -(-n // BLOCK)
    ms, vs = (torch.randint(118, 126, (blocks,), generator=g, dtype=torch.uint8) for _ in range(2))
    for off in (0, 1):
        def place(t):
            buf = torch.zeros(t.numel() + off, dtype=t.dtype, device=dev)
            buf[off:] = t.to(dev)
            return buf[off:]

        got = ops.adamw_moments(place(m), place(v), place(ms), place(vs), dtype=dtype)
        for x, code, scale, which in ((got[0], m, ms, "m"), (got[1], v, vs, "v")):
            want = decode(code, scale, which).to(dtype).cpu()
            assert torch.equal(torch.isnan(x.cpu()), torch.isnan(want))
            assert torch.equal(torch.nan_to_num(x.cpu()), torch.nan_to_num(want))


def test_device_counter_and_captured_steps(dev):
    """adamw_advance counts as the host would; a captured norm + advance + step replayed with new gradients and
    a new learning rate gives the eager result, a bad gradient's replay changes nothing and does not count."""
    from unirl_amd import ops

    lr = torch.tensor(1e-3, device=dev)
    hyper = {k: HYPER[k] for k in ("betas", "eps")}
    for bits in (32, 8):
        _, D = make([700, 5000], torch.bfloat16, torch.bfloat16, bits, True, 8, dev)
        _, E = make([700, 5000], torch.bfloat16, torch.bfloat16, bits, True, 8, dev)
        count, control = torch.zeros((), dtype=torch.int64, device=dev), torch.zeros(32, dtype=torch.uint8, device=dev)

        def step():
            norm = ops.grad_norm([d["grad"] for d in D])
            ops.adamw_advance(count, control, lr=lr, betas=HYPER["betas"], weight_decay=0.1, seed=4, grad_norm=norm,
                              max_norm=0.1, skip_nonfinite=True)
            apply(D, hyper, control=control)

        def compare():
            torch.cuda.synchronize()
            for d, e in zip(D, E):
                for k in set(d) - {"grad"}:  # an input, and NaN equals nothing
                    assert torch.equal(d[k], e[k]), (bits, k)

        step()
        taken = 1
        # the rate on the device is the fp32 number next to 1e-3: the other side is asked for the same one
        apply(E, hyper, lr=float(lr), weight_decay=0.1, step=1, seed=4, grad_norm=ops.grad_norm([e["grad"] for e in E]), max_norm=0.1)
        compare()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for i in range(5):
            bad = i == 2
            rate = 1e-3 / (i + 1)
            lr.fill_(rate)
            for d, e in zip(D, E):
                e["grad"].normal_()
                if bad:
                    e["grad"][3] = float("nan")
                d["grad"].copy_(e["grad"])
            graph.replay()
            if not bad:
                taken += 1
                apply(E, hyper, lr=float(lr), weight_decay=0.1, step=taken, seed=4,
                      grad_norm=ops.grad_norm([e["grad"] for e in E]), max_norm=0.1)
            compare()
            assert int(count) == taken
        lr.fill_(1e-3)


def test_streams_and_graphs_do_not_share_scratch(dev):
    """Norms of different gradients on two streams at once, and of two graphs replayed in turn with eager
    calls between: each gives the value of its own input."""
    from unirl_amd import ops

    sets = [[torch.randn(3_000_001 + 7 * k + i, device=dev) * (k + 1) for i in range(5)] for k in range(2)]
    want = [float(ops.grad_norm(s)) for s in sets]
    assert want[0] != want[1]
    streams = [torch.cuda.Stream(dev) for _ in sets]
    got = [[], []]
    torch.cuda.synchronize()
    for _ in range(10):
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[k].append(ops.grad_norm(sets[k]))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(float(v) == want[k] for v in got[k])
    graphs, outs = [], []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.grad_norm(s))
        graphs.append(graph)
    for _ in range(4):
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                outs[k].zero_()
                graphs[k].replay()
        torch.cuda.synchronize()
        assert [float(v) for v in outs] == want
        assert float(ops.grad_norm(sets[0] + sets[1])) > max(want)


def test_first_step_that_is_skipped(dev):
    """A bad gradient in the first step: nothing is written, nothing counted; the next step is step 1."""
    from unirl_amd.train import AdamW

    for bits in (32, 8):
        ours, twin = model(torch.bfloat16, dev), model(torch.bfloat16, dev)
        kw = dict(lr=1e-2, state_bits=bits, master_weights=True)
        a, b = AdamW(ours, capturable=True, skip_nonfinite=True, **kw), AdamW(twin, **kw)
        set_grads(ours, 0)
        ours[1].grad[3] = float("inf")
        before = [p.detach().clone() for p in ours]
        a.step()
        assert math.isinf(float(a.grad_norm)) and int(a.param_groups[0]["step"]) == 0
        assert all(torch.equal(p, q) for p, q in zip(ours, before))
        for k in range(2):
            set_grads(ours, k)
            set_grads(twin, k)
            a.step()
            b.step()
        assert all(torch.equal(p, q) for p, q in zip(ours, twin)) and int(a.param_groups[0]["step"]) == 2


def test_a_step_between_forward_and_backward_is_noticed(dev):
    from unirl_amd import models
    from unirl_amd.train import AdamW

    w = torch.nn.Parameter(torch.ones(64, device=dev))
    x = torch.randn(5, 64, device=dev, requires_grad=True)
    y = models.rms_norm(x, w)
    w.grad = torch.ones_like(w)
    AdamW([w]).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_refusals(dev):
    from unirl_amd import ops

    def t(n=8, dtype=torch.float32):
        return torch.zeros(n, dtype=dtype, device=dev)

    base = dict(lr=1e-3, step=1)
    p = t()
    bad = [
        lambda: ops.adamw_step([p, p], [t(), t()], [t(), t()], [t(), t()], **base),  # one tensor twice
        lambda: ops.adamw_step([t()], [t(9)], [t()], [t()], **base),
        lambda: ops.adamw_step([t()], [t()], [t(dtype=torch.uint8)], [t()], **base),
        lambda: ops.adamw_step([t()], [t()], [t()], [t(9)], **base),
        lambda: ops.adamw_step([t(16)[::2]], [t()], [t()], [t()], **base),
        lambda: ops.adamw_step([t(), t(dtype=torch.bfloat16)], [t(), t()], [t(), t()], [t(), t()], **base),
        lambda: ops.adamw_step([t()], [t()], [t()], [t()], masters=[t()], **base),
        lambda: ops.adamw_step([t()], [t()], [t()], [t()], lr=1e-3),
        lambda: ops.adamw_step([t()], [t()], [t()], [t()], lr=1e-3, step=0),
        lambda: ops.adamw_step([t()], [t()], [t()], [t()], max_norm=1.0, **base),
        lambda: ops.adamw_step([t()], [t()], [t()], [t()], grad_norm=t(2), max_norm=1.0, **base),
        lambda: ops.adamw_step([t()], [t()], [t()], [t()], grad_norm=t(1), max_norm=-1.0, **base),
        lambda: ops.adamw_step([t()], [t()], [t()], [t()], grad_norm=t(1), max_norm=float("nan"), **base),
        lambda: ops.adamw_step([t()], [t()], [t()], [t()], control=t(32, torch.uint8), **base),
        lambda: ops.adamw_step([t()], [t()], [t()], [t()], control=t(31, torch.uint8)),
        lambda: ops.adamw_step([t()], [t()], [t(dtype=torch.uint8)], [t(dtype=torch.uint8)], exp_avg_scales=[t(2, torch.uint8)],
                               exp_avg_sq_scales=[t(1, torch.uint8)], **base),
        lambda: ops.adamw_step([t()], [t()], [t(dtype=torch.uint8)], [t(dtype=torch.uint8)], exp_avg_scales=[t(1, torch.uint8)],
                               exp_avg_sq_scales=[t(1, torch.uint8)], index_bases=[100], **base),
        lambda: ops.adamw_advance(t(1), t(32, torch.uint8), lr=1e-3),
        lambda: ops.adamw_advance(t(1, torch.int64), t(32, torch.uint8), lr=t(2)),
        lambda: ops.adamw_moments(t(300, torch.uint8), t(300, torch.uint8), t(1, torch.uint8), t(2, torch.uint8)),
        lambda: ops.adamw_moments(t(300), t(300), t(2, torch.uint8), t(2, torch.uint8)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(TypeError):
        ops.adamw_step([t()], [t(dtype=torch.bfloat16)], [t()], [t()], **base)
    with pytest.raises(TypeError):
        ops.grad_norm([t(dtype=torch.float64)])
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------ the optimizer
def model(dtype, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter((torch.randn(s, generator=g) * 0.1).to(dtype).to(dev)) for s in ((33, 20), (20,), (7, 3, 5), ())]


def set_grads(params, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    for p in params:
        p.grad = (torch.randn(p.shape, generator=g) * scale).to(p.dtype).to(p.device)


def test_optimizer_follows_torch_adamw(dev):
    """fp32, two groups, clipping, a parameter without a gradient in some steps: torch's AdamW in 64 bits.
    Per step p moves by at most about lr with a relative error of 30 u, and rounds by 3 u |p| (the bounds
    above): 10 steps stay below 10 (30 u lr + 3 u (|p| + lr))."""
    from unirl_amd.train import AdamW

    ours, ref = model(torch.float32, dev), [torch.nn.Parameter(p.detach().double().cpu()) for p in model(torch.float32, dev)]

    def groups(ps):
        return [dict(params=ps[:2], lr=1e-2), dict(params=ps[2:], weight_decay=0.0)]

    a = AdamW(groups(ours), lr=3e-3, betas=(0.9, 0.95), weight_decay=0.1, max_grad_norm=1.5)
    b = torch.optim.AdamW(groups(ref), lr=3e-3, betas=(0.9, 0.95), weight_decay=0.1)
    for step in range(10):
        set_grads(ours, step)
        for p, q in zip(ours, ref):
            q.grad = p.grad.double().cpu()
        if step % 3 == 1:
            ours[1].grad = ref[1].grad = None
        version = ours[0]._version
        a.step()
        assert ours[0]._version > version
        norm = torch.nn.utils.clip_grad_norm_(ref, 1.5)
        b.step()
        assert abs(float(a.grad_norm) - float(norm)) <= 1.01 * U * float(norm)
    for p, q in zip(ours, ref):
        off = (p.detach().double().cpu() - q.detach()).abs()
        assert bool((off <= 10 * U * (30 * 1e-2 + 3 * (q.detach().abs() + 1e-2))).all())


@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_state_round_trip(dev, bits, capturable):
    """Saved, loaded into a new optimizer and stepped on: the same bytes as without the interruption."""
    import io

    from unirl_amd.train import AdamW

    kw = dict(lr=1e-2, state_bits=bits, master_weights=True, max_grad_norm=1.0, capturable=capturable, seed=3)
    ours, twin = model(torch.bfloat16, dev), model(torch.bfloat16, dev)
    a = AdamW(ours, **kw)
    for step in range(3):
        set_grads(ours, step)
        a.step()
    buf = io.BytesIO()
    torch.save(a.state_dict(), buf)
    buf.seek(0)
    b = AdamW(twin, **kw)
    b.load_state_dict(torch.load(buf, weights_only=True))
    for p, q in zip(ours, twin):
        q.data.copy_(p.data)
    for step in range(3, 6):
        set_grads(ours, step)
        set_grads(twin, step)
        a.step()
        b.step()
    for p, q in zip(ours, twin):
        assert torch.equal(p, q)
        assert set(a.state[p]) == set(b.state[q])
        for k, v in a.state[p].items():
            w = b.state[q][k]
            assert torch.equal(v, w) and v.dtype == w.dtype if isinstance(v, torch.Tensor) else v == w, k
        m, v = b.moments(q)
        assert m.dtype == v.dtype == torch.float32 and m.shape == q.shape and bool((v >= 0).all())
    other = AdamW(model(torch.bfloat16, dev), state_bits=40 - bits)
    with pytest.raises(ValueError, match="saved moments"):
        other.load_state_dict(a.state_dict())


def test_optimizer_copies_groups_and_schedulers(dev):
    """A deep copy steps like the original; a scheduler's rate is used; a group added later joins in."""
    import copy

    from unirl_amd.train import AdamW

    ours = model(torch.float32, dev)
    a = AdamW(ours[:2], lr=1e-2, state_bits=8, max_grad_norm=1.0, capturable=True, skip_nonfinite=True)
    rate = torch.optim.lr_scheduler.LambdaLR(a, lambda k: 1.0 / (k + 1))
    set_grads(ours, 0)
    a.step()
    rate.step()
    a.add_param_group(dict(params=ours[2:], state_bits=32))
    set_grads(ours, 1)
    a.step()
    twin = copy.deepcopy({"opt": a, "params": ours})
    b, theirs = twin["opt"], twin["params"]
    assert (b.max_grad_norm, b.skip_nonfinite, b.capturable) == (1.0, True, True)
    set_grads(ours, 2)
    set_grads(theirs, 2)
    before = [p.detach().clone() for p in ours]
    a.step()
    b.step()
    for p, q, old in zip(ours, theirs, before):
        assert torch.equal(p, q) and not torch.equal(p, old)
    assert [int(g["step"]) for g in b.param_groups] == [3, 2]
    bases = [a.state[p]["index_base"] for p in ours]
    assert len(set(bases)) == len(bases) and all(x % 256 == 0 for x in bases)


def test_master_weights_keep_small_updates(dev):
    """Updates of a fiftieth of a bf16 unit: 100 of them move the parameter with a master, none without."""
    from unirl_amd.train import AdamW

    for master in (True, False):
        p = torch.nn.Parameter(torch.ones(64, device=dev, dtype=torch.bfloat16))
        opt = AdamW([p], lr=2.0**-7 / 50, weight_decay=0.0, betas=(0.0, 0.0), master_weights=master)
        for _ in range(100):
            p.grad = torch.full_like(p, -1.0)
            opt.step()
        # each step adds lr (m / sqrt(v) = -1): 1 + 2 * 2^-7
        assert bool((p == (1 + 2 * 2.0**-7 if master else 1.0)).all())


def test_masters_follow_written_parameters_on_request(dev):
    from unirl_amd.train import AdamW

    p = torch.nn.Parameter(torch.ones(8, device=dev, dtype=torch.bfloat16))
    opt = AdamW([p], lr=0.0, weight_decay=0.0, master_weights=True)
    p.grad = torch.ones_like(p)
    opt.step()
    with torch.no_grad():
        p.fill_(3.0)
    opt.step()
    assert bool((p == 1.0).all())  # the master leads
    with torch.no_grad():
        p.fill_(3.0)
    opt.refresh_masters()
    opt.step()
    assert bool((p == 3.0).all())


def test_captured_optimizer(dev):
    from unirl_amd.train import AdamW

    ours, twin = model(torch.bfloat16, dev), model(torch.bfloat16, dev)
    kw = dict(lr=1e-2, state_bits=8, master_weights=True, max_grad_norm=1.0, seed=3)
    a, b = AdamW(ours, capturable=True, skip_nonfinite=True, **kw), AdamW(twin, **kw)
    set_grads(ours, 0)
    set_grads(twin, 0)
    grads = [p.grad for p in ours]
    a.step()
    b.step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        a.step()
    for step in range(1, 6):
        set_grads(twin, step)
        for g, q in zip(grads, twin):
            g.copy_(q.grad)
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        for p, q in zip(ours, twin):
            assert torch.equal(p, q), step
    # a captured step without a device count, or before there is state, is refused
    for opt in (b, AdamW(model(torch.float32, dev), capturable=True)):
        for group in opt.param_groups:
            set_grads(group["params"], 1)
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="AdamW"):
            with torch.cuda.graph(graph):
                opt.step()
        torch.cuda.synchronize()


def test_policy_update_end_to_end(dev):
    """Final norm, head, log-prob, GRPO loss with its gradient (at ratio 1, where it is the policy gradient), global
    norm and clipped step in one run, against the same chain in 64 bits on the CPU; the bf16 chain's gradients are compared at bf16's resolution of
    their largest terms (2^-7 of the column's largest: logits, norm output and gradient are rounded to
    2^-8 each), the step with the chain's own gradients at the step's bounds."""
    from unirl_amd import models
    from unirl_amd.algorithms import fused_token_loss_backward
    from unirl_amd.train import AdamW

    g = torch.Generator().manual_seed(1)
    B, T, D, V = 4, 48, 128, 512
    hidden = torch.randn(B, T, D, generator=g).bfloat16()
    tokens = torch.randint(0, V, (B, T), generator=g)
    adv = torch.randn(B, generator=g)
    norm = torch.nn.RMSNorm(D, eps=1e-6, dtype=torch.bfloat16)
    head = torch.nn.Linear(D, V, bias=False, dtype=torch.bfloat16)
    with torch.no_grad():
        norm.weight.copy_(1 + 0.1 * torch.randn(D, generator=g))
        head.weight.copy_(torch.randn(V, D, generator=g) / math.sqrt(D))
    W, N = head.weight.detach().double().requires_grad_(True), norm.weight.detach().double().requires_grad_(True)
    X = hidden.double()
    Y = X / torch.sqrt((X * X).mean(-1, keepdim=True) + 1e-6) * N
    logp = torch.log_softmax(Y @ W.t(), -1).gather(-1, tokens[..., None])[..., 0]
    exact = torch.autograd.grad(-(logp * adv[:, None]).mean(), [W, N])

    norm, head = norm.to(dev), head.to(dev)
    params = [head.weight, norm.weight]
    opt = AdamW(params, lr=1e-3, state_bits=8, master_weights=True, max_grad_norm=1e-3)
    new = models.chunked_replay_logp(head, hidden.to(dev), tokens.to(dev), final_norm=norm)
    fused_token_loss_backward("grpo", new, new.detach(), adv.to(dev), loss_scale=1.0,
                              lengths=torch.full((B,), T, device=dev, dtype=torch.int64))
    for p, e in zip(params, exact):
        off = (p.grad.double().cpu() - e).abs().max()
        assert float(off) <= 2.0**-7 * float(e.abs().max()), float(off / e.abs().max())
    before = [p.detach().clone() for p in params]
    grads = [p.grad.double().cpu() for p in params]
    opt.step()
    total = math.sqrt(sum(float((x * x).sum()) for x in grads))
    assert abs(float(opt.grad_norm) - total) <= 1.01 * U * total
    c = min(1.0, 1e-3 / (total + 1e-6))
    for p, b, gr in zip(params, before, grads):
        t = dict(param=b.cpu(), master=b.float().cpu(), grad=gr, m=torch.zeros_like(gr), v=torch.zeros_like(gr))
        want, _, _ = reference(t, dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, step=1), c, 0)
        check(p.detach(), want["param"], "parameter")
        check(opt.state[p]["master"], want["master"], "master")

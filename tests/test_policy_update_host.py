"""CPU-only checks of the norm, gradient-norm and AdamW entry points: argument errors come back as
statuses before anything is launched, the structures are laid out as the header declares them, and the
Python layer refuses what the kernels do not handle."""

import ctypes
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent
FAKE = 0x10000  # never dereferenced: every call below is refused, or has nothing to do


def _desc(N, **over):
    f = dict(x=FAKE, dtype=N.BF16, x_group_stride=0, x_row_stride=64, groups=1, rows=4, D=64, gain=FAKE, bias=None,
             gain_dtype=N.BF16, gain_group_stride=0, bias_group_stride=0, gain_offset=0.0, center=1, eps=1e-5, mean=FAKE,
             rstd=FAKE)
    f.update(over)
    return N.NormDesc(**f)


@pytest.mark.parametrize("over,status", [
    (dict(dtype=7), -3), (dict(gain_dtype=9), -3), (dict(rows=-1), -2), (dict(groups=-1), -2), (dict(D=0), -2),
    (dict(D=32769), -6), (dict(x=None), -1), (dict(x=FAKE + 1), -5), (dict(gain=FAKE + 1), -5), (dict(mean=FAKE + 2), -5),
    (dict(x_row_stride=-64), -2), (dict(gain_group_stride=-1), -2), (dict(rows=0), 0), (dict(groups=0, x=None), 0),
])
def test_norm_forward_refusals(built_lib, over, status):
    from unirl_amd import _native as N

    assert N.lib().unirl_layer_norm_fwd(ctypes.byref(_desc(N, **over)), FAKE, None) == status


def test_norm_refuses_missing_operands(built_lib):
    from unirl_amd import _native as N

    L = N.lib()
    assert L.unirl_layer_norm_fwd(None, FAKE, None) == -1
    assert L.unirl_layer_norm_fwd(ctypes.byref(_desc(N)), None, None) == -1
    assert L.unirl_layer_norm_fwd(ctypes.byref(_desc(N)), FAKE + 1, None) == -5

    def bwd(desc=None, dy=FAKE, dys=64, dx=FAKE, dgain=FAKE, dbias=None, per_group=0, scratch=FAKE, nbytes=1 << 40):
        return L.unirl_layer_norm_bwd(ctypes.byref(desc or _desc(N)), dy, 0, dys, dx, dgain, dbias, per_group, scratch, nbytes,
                                      None)

    assert bwd(dy=None) == -1
    assert bwd(_desc(N, rstd=None)) == -1
    assert bwd(_desc(N, mean=None)) == -1
    assert bwd(dys=-1) == -2
    assert bwd(dy=FAKE + 1) == -5
    assert bwd(dx=FAKE + 1) == -5
    assert bwd(dgain=FAKE + 1) == -5
    assert bwd(scratch=None) == -4
    assert bwd(nbytes=int(L.unirl_layer_norm_bwd_scratch_bytes(1, 4, 64)) - 1) == -4
    assert bwd(scratch=FAKE + 4) == -5
    assert bwd(_desc(N, groups=65536), per_group=1) == -6
    assert bwd(dx=None, dgain=None) == 0  # nothing is wanted


def test_norm_scratch_grows_with_columns_and_is_bounded_in_rows(built_lib):
    from unirl_amd import _native as N

    size = N.lib().unirl_layer_norm_bwd_scratch_bytes
    assert size(0, 5, 8) == size(1, 0, 8) == size(1, 5, 0) == size(1, 5, 40000) == 0
    assert size(1, 1, 8) >= 2 * 4 * 8
    assert size(1, 1 << 40, 4096) <= 2 * 4 * 4096 * 4096  # a bounded number of partial rows


def _adamw(N, tensors=None, n=None, **over):
    f = dict(param_dtype=N.F32, grad_dtype=N.F32, state_bits=32, use_master=0, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8,
             weight_decay=0.0, step=1, seed=0, grad_norm=None, max_norm=-1.0, skip_nonfinite=0, control=None)
    f.update(over)
    t = tensors or [dict()]
    arr = (N.AdamwTensor * len(t))()
    for i, d in enumerate(t):
        g = dict(param=FAKE, grad=FAKE, exp_avg=FAKE, exp_avg_sq=FAKE, master=None, exp_avg_scale=None, exp_avg_sq_scale=None,
                 numel=4, index_base=0)
        g.update(d)
        arr[i] = N.AdamwTensor(**g)
    q = N.AdamwParams(**f)
    return N.lib().unirl_adamw_step(ctypes.byref(arr), len(t) if n is None else n, ctypes.byref(q), None)


def test_adamw_refusals(built_lib):
    from unirl_amd import _native as N

    assert _adamw(N, param_dtype=5) == -3
    assert _adamw(N, grad_dtype=N.BF16) == -3  # fp32 parameters have fp32 gradients
    assert _adamw(N, param_dtype=N.BF16, grad_dtype=N.F16) == -3
    assert _adamw(N, state_bits=16) == -3
    assert _adamw(N, use_master=1) == -3
    assert _adamw(N, step=0) == -2
    assert _adamw(N, beta1=1.0) == -2
    assert _adamw(N, beta2=-0.1) == -2
    assert _adamw(N, beta2=float("nan")) == -2
    assert _adamw(N, n=-1) == -2
    assert _adamw(N, [dict(numel=-1)]) == -2
    assert _adamw(N, [dict(index_base=-256)]) == -2
    assert _adamw(N, [dict(param=None)]) == -1
    assert _adamw(N, [dict(exp_avg_sq=None)]) == -1
    assert _adamw(N, state_bits=8) == -1  # no scales
    assert _adamw(N, [dict(exp_avg_scale=FAKE, exp_avg_sq_scale=FAKE, index_base=128)], state_bits=8) == -5
    assert _adamw(N, [dict(param=FAKE + 2)]) == -5
    assert _adamw(N, [dict(exp_avg=FAKE + 1)]) == -5
    assert _adamw(N, param_dtype=N.BF16, grad_dtype=N.BF16, use_master=1) == -1
    assert _adamw(N, grad_norm=FAKE + 1) == -5
    assert _adamw(N, [dict(numel=1 << 60)]) == -6
    # a bad entry behind good ones is found before the first launch
    assert _adamw(N, [dict()] * 60 + [dict(grad=None)]) == -1
    assert _adamw(N, n=0) == 0
    assert _adamw(N, [dict(numel=0, param=None, grad=None)]) == 0
    L = N.lib()
    assert L.unirl_adamw_step(None, 1, ctypes.byref(N.AdamwParams()), None) == -1
    assert L.unirl_adamw_step(None, 0, None, None) == -1
    assert L.unirl_adamw_advance(None, FAKE, 1e-3, None, 0.9, 0.9, 0.0, 0, None, -1.0, 0, None) == -1
    assert L.unirl_adamw_advance(FAKE + 4, FAKE, 1e-3, None, 0.9, 0.9, 0.0, 0, None, -1.0, 0, None) == -5
    assert L.unirl_adamw_advance(FAKE, FAKE, 1e-3, None, 0.9, 1.0, 0.0, 0, None, -1.0, 0, None) == -2
    assert L.unirl_adamw_moments(None, FAKE, FAKE, FAKE, 4, FAKE, FAKE, N.F32, None) == -1
    assert L.unirl_adamw_moments(FAKE, FAKE, FAKE, FAKE, -4, FAKE, FAKE, N.F32, None) == -2
    assert L.unirl_adamw_moments(FAKE, FAKE, FAKE, FAKE, 4, FAKE, FAKE, 8, None) == -3
    assert L.unirl_adamw_moments(FAKE, FAKE, FAKE, FAKE, 4, FAKE + 2, FAKE, N.F32, None) == -5
    assert L.unirl_adamw_moments(None, None, None, None, 0, None, None, N.F32, None) == 0


def test_grad_norm_refusals(built_lib):
    from unirl_amd import _native as N

    def call(ptrs, numels, codes, n=None, out=FAKE, ws=FAKE, nbytes=1 << 30):
        k = len(ptrs)
        return N.lib().unirl_grad_norm(ctypes.byref((ctypes.c_void_p * max(k, 1))(*ptrs)), ctypes.byref((ctypes.c_int64 * max(k, 1))(*numels)),
                                       ctypes.byref((ctypes.c_int * max(k, 1))(*codes)), k if n is None else n, out, ws, nbytes, None)

    assert call([FAKE], [4], [0], out=None) == -1
    assert call([None], [4], [0]) == -1
    assert call([FAKE], [-4], [0]) == -2
    assert call([FAKE], [4], [3]) == -3
    assert call([FAKE + 2], [4], [0]) == -5
    assert call([FAKE], [4], [0], out=FAKE + 2) == -5
    assert call([FAKE], [4], [0], ws=None) == -4
    assert call([FAKE], [4], [0], nbytes=64) == -4
    assert call([FAKE], [4], [0], ws=FAKE + 8) == -5
    assert call([FAKE], [4], [0], n=-1) == -2
    assert call([FAKE], [1 << 62], [0]) == -6


def test_structures_match_the_header(built_lib, tmp_path):
    """Sizes and offsets of the three structures as a C compiler lays them out."""
    from unirl_amd import _native as N

    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler on this host")
    pairs = [("unirl_norm_desc", N.NormDesc), ("unirl_adamw_tensor", N.AdamwTensor), ("unirl_adamw_params", N.AdamwParams)]
    lines = [f'printf("%zu ", sizeof(struct {c}));' + "".join(f'printf("%zu ", offsetof(struct {c}, {f[0]}));' for f in t._fields_)
             for c, t in pairs]
    src = tmp_path / "l.c"
    src.write_text('#include <stdio.h>\n#include "unirl_hip.h"\nint main(void){' + "".join(lines)
                   + 'printf("%d", UNIRL_ADAMW_CONTROL_BYTES);return 0;}\n')
    subprocess.run([cc, "-std=c99", "-I", str(ROOT / "include"), "-o", str(tmp_path / "l"), str(src)], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for _, t in pairs:
        want += [ctypes.sizeof(t)] + [getattr(t, f[0]).offset for f in t._fields_]
    assert got == want + [N.ADAMW_CONTROL_BYTES]


def test_python_layer_refuses_what_the_kernels_do_not_handle(built_lib):
    from unirl_amd import models, ops, train

    x, w = torch.randn(3, 8), torch.ones(8)
    for call in (
        lambda: ops.layer_norm(x, w), lambda: models.rms_norm(x, w), lambda: models.layer_norm(x),
        lambda: models.modulated_layer_norm(x, x, x), lambda: ops.grad_norm([x]),
        lambda: ops.adamw_step([x], [x], [x], [x], lr=1e-3, step=1),
    ):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
    with pytest.raises(ValueError, match="at least one tensor"):
        ops.grad_norm([])
    with pytest.raises(ValueError, match="entries"):
        ops.adamw_step([x], [x], [x], [], lr=1e-3, step=1)
    with pytest.raises(ValueError, match="exp_avg_sq_scales"):
        ops.adamw_step([x], [x], [x], [x], lr=1e-3, step=1, exp_avg_scales=[x])
    with pytest.raises(ValueError, match="betas"):
        ops.adamw_step([x], [x], [x], [x], lr=1e-3, step=1, betas=(0.9, 1.0))
    ops.adamw_step([], [], [], [], lr=1e-3, step=1)  # nothing to do
    with pytest.raises(ValueError, match="modulated_layer_norm"):
        models.layer_norm(x, torch.ones(3, 8))
    with pytest.raises(ValueError, match="scale"):
        models.modulated_layer_norm(x, torch.ones(8), torch.ones(3, 8))

    p = torch.nn.Parameter(torch.randn(4, 6))
    for kw in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-0.1), dict(state_bits=4),
               dict(max_grad_norm=-1.0), dict(skip_nonfinite=True), dict(lr=torch.tensor(1e-3))):
        with pytest.raises(ValueError):
            train.AdamW([p], **kw)
    with pytest.raises(ValueError, match="contiguous"):
        train.AdamW([torch.nn.Parameter(torch.randn(4, 6).t())])
    with pytest.raises(TypeError):
        train.AdamW([torch.nn.Parameter(torch.randn(4, dtype=torch.float64))])
    opt = train.AdamW([p])
    opt.step()  # no gradient: nothing to do
    p.grad = torch.ones_like(p)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        opt.step()


def test_dither_hash_is_a_fair_coin_per_bit():
    """The mixing function of the stochastic rounding, restated: every input bit flips every output bit
    in half of the cases.  65 536 samples have a standard deviation of 0.00195; over the 1024 pairs the
    largest deviation of a fair coin stays below 5 of them."""
    import numpy as np

    source = (ROOT / "unirl_amd" / "csrc" / "optim.hip").read_text()
    body = re.search(r"uint32_t mix32\(uint32_t x\) \{(.*?)\n\}", source, flags=re.S).group(1)
    shifts = [int(s) for s in re.findall(r">> (\d+)", body)]
    mults = [int(m, 16) for m in re.findall(r"\*= (0x[0-9A-F]+)u", body)]
    assert (len(shifts), len(mults)) == (3, 2)

    def mix(x):
        x = x ^ (x >> np.uint64(shifts[0]))
        x = (x * np.uint64(mults[0])) & np.uint64(0xFFFFFFFF)
        x = x ^ (x >> np.uint64(shifts[1]))
        x = (x * np.uint64(mults[1])) & np.uint64(0xFFFFFFFF)
        return x ^ (x >> np.uint64(shifts[2]))

    x = np.random.RandomState(2).randint(0, 1 << 32, 65536, dtype=np.uint64)
    h = mix(x)
    worst = 0.0
    for b in range(32):
        d = h ^ mix(x ^ np.uint64(1 << b))
        flips = [float(((d >> np.uint64(o)) & np.uint64(1)).mean()) for o in range(32)]
        worst = max(worst, max(abs(f - 0.5) for f in flips))
    assert worst < 5 * 0.5 / 256

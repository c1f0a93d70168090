"""AdamW over lists around the number of tensors that one launch takes: 90 (fp32 moments), 76 (with a master), 58
(8-bit moments) and 52 (with a master).  No tensor is empty, so that the next launch's table, scales and dither
positions among it, is filled anew from the first entry on."""

import pytest
import torch

from tests.test_gpu_optim import HYPER, apply, check, check_codes, dither, make, reference

pytestmark = pytest.mark.gpu

COUNTS = [51, 52, 53, 57, 58, 59, 75, 76, 77, 89, 90, 91, 181]


@pytest.mark.parametrize("count", COUNTS)
@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_lists_around_a_launch(dev, bits, master, count):
    sizes = [1 + (i * 37) % 300 for i in range(count)]
    T, D = make(sizes, torch.bfloat16, torch.bfloat16, bits, master, count, dev)
    apply(D, HYPER, seed=11)
    base = 0
    for i, (t, d) in enumerate(zip(T, D)):
        want, m, v = reference(t, HYPER, 1.0, base)
        for name in want:
            check(d[name], want[name], f"{name} of tensor {i}")
        if bits == 8:
            wm, wv = dither(m.numel(), base, 11, HYPER["step"])
            check_codes(d["m"], d["ms"], m, wm, "m", f"m of tensor {i}")
            check_codes(d["v"], d["vs"], v, wv, "v", f"v of tensor {i}")
        base += -(-m.numel() // 256) * 256

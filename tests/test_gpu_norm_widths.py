"""Values and gradients of the norms at widths that between them reach every kernel: each number of elements a
lane holds, each width of workgroup, forward and backward, in vectors and one by one
(``test_norm_shapes_host.py`` counts that none is missing).

The bounds are those of ``test_gpu_norm.py`` with its sums' longest chain corrected: a lane of the forward holds up
to 64 elements of a row that belongs to one wavefront, 64 + 6 = 70 additions (in a workgroup 32 + 6 + 16 = 54, and
no more than 54 in the backward).  The mean is then off by 73 u A instead of 57 u A, the root by 73 u A s + 43 u
instead of 57 u A s + 35 u, xh's own rounding by 48 u instead of 40 u: every part of a bound but the final
rounding grows by a factor of at most 73 / 57 < 1.3.
"""

import pytest
import torch

from tests.test_gpu_norm import DTYPES, TINY, check, half, make, reference, run

pytestmark = pytest.mark.gpu

WIDTHS = [16, 120, 136, 264, 500, 1032, 1100, 1336, 1536, 1800, 2049, 2504, 2568, 3000, 3080, 3333, 3584, 4095, 4096, 4104, 5000, 5120, 6144, 6145,
          6152, 7000, 8201, 9000, 12289, 12296, 16383, 16392, 16400, 16401, 24577, 24584, 28671]


def widened(want, dtype):
    value, bound = want
    last = half(dtype) * value.abs() * 1.01 + TINY[dtype]
    return value, 1.3 * (bound - last) + last


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("kind", ["layer", "rms", "mod"])
def test_every_width_of_kernel(dev, kind, D, dtype):
    x, w, b, dy = make((2, 6, D) if kind == "mod" else (11, D), dtype, D + 1, kind == "mod", bias=kind != "rms")
    want = reference(x, w, b, dy, 1e-5, kind == "rms", 1.0 if kind == "mod" else 0.0)
    got = run(x, w, b, dy, 1e-5, kind, dev)
    for name in want:
        check(got[name], widened(want[name], dtype), f"{kind} {D} {dtype} {name}")

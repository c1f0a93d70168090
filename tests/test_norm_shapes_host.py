"""CPU-only: the widths whose values the GPU tests compare reach every kernel that the norms' launches choose."""

import re
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def shapes(tmp_path_factory):
    """``norm_shape`` for every width, compiled from the kernels' source: {(bytes of an element, vectors,
    backward): [(lanes, vec, elems, threads) of D = 1, 2, ...]}."""
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no C++ compiler on this host")
    source = (ROOT / "unirl_amd" / "csrc" / "norm.hip").read_text()
    struct = re.search(r"struct NormShape \{.*?\n\};", source, flags=re.S).group(0)
    function = re.search(r"static NormShape norm_shape\(.*?\n\}", source, flags=re.S).group(0)
    rows = re.findall(r"constexpr int (kNorm(?:Fwd|Bwd)Rows) = (\d+);", source)
    limit = re.search(r"constexpr int kNormMaxDim = (\d+);", source).group(1)
    tmp = tmp_path_factory.mktemp("shapes")
    (tmp / "s.cpp").write_text(
        "#include <cstdint>\n#include <cstdio>\nenum { UNIRL_F32, UNIRL_BF16 };\nconstexpr int kWave = 64;\n"
        "static size_t dtype_size(int d) { return d == UNIRL_F32 ? 4 : 2; }\n"
        + "".join(f"constexpr int {k} = {v};\n" for k, v in rows) + struct + "\n" + function
        + "\nint main() { for (int64_t D = 1; D <= %s; ++D) for (int t = 0; t < 2; ++t) for (int v = 0; v < 2; ++v)"
          " for (int b = 0; b < 2; ++b) { const NormShape S = norm_shape(D, t, v, b);"
          ' printf("%%d %%d %%d %%d\\n", S.lanes, S.vec, S.elems, S.threads); } }\n' % limit)
    subprocess.run([cxx, "-O1", "-std=c++17", "-o", str(tmp / "s"), str(tmp / "s.cpp")], check=True)
    out = subprocess.run([str(tmp / "s")], check=True, capture_output=True, text=True).stdout.split()
    flat = [tuple(int(v) for v in out[i : i + 4]) for i in range(0, len(out), 4)]
    keys = [(size, v, b) for size in (4, 2) for v in (False, True) for b in (False, True)]
    return {key: flat[i :: len(keys)] for i, key in enumerate(keys)}


def kernels(shapes):
    """{kernel: widths that run it}: what a template's arguments tell apart."""
    found = {}
    for (size, vectors, backward), per_width in shapes.items():
        for D, (lanes, vec, elems, threads) in enumerate(per_width, 1):
            if vectors != (D % (16 // size) == 0):
                continue  # a dense tensor of this width goes the other way
            limits = (512, 768, 1024) if backward and elems <= 16 else ((1024,) if backward else (512, 1024))
            bound = 0 if lanes else next(t for t in limits if threads <= t)
            found.setdefault((size, vec, backward, lanes, elems, bound), []).append(D)
    return found


def test_every_kernel_has_a_tested_width(shapes):
    from tests.test_gpu_norm import DIMS
    from tests.test_gpu_norm_widths import WIDTHS

    tested = set(DIMS) | set(WIDTHS)
    missing = {k: (w[0], w[-1]) for k, w in kernels(shapes).items() if not tested & set(w)}
    assert not missing, missing


def test_every_row_fits_its_threads(shapes):
    """Lanes times elements cover the row, inside the widths that are launched; and no kernel holds more than the
    tests' bounds count on (64 elements a lane forward, 32 backward)."""
    for (size, vectors, backward), per_width in shapes.items():
        for D, (lanes, vec, elems, threads) in enumerate(per_width, 1):
            if vectors and D % (16 // size):
                continue
            width = lanes or threads
            assert width * elems >= D and elems % vec == 0 and threads <= 1024, (size, vectors, backward, D)
            assert elems <= (64 if lanes else 32) and (not backward or elems <= 32), (size, vectors, backward, D)

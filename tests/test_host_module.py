"""The C++ module that reads tensors names the ABI that it was compiled against."""

import re
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


def test_host_module_reports_its_own_abi_version(built_lib, tmp_path):
    """Loaded beside a library of another version (a stand-in with the same symbols), the module still
    reports the header's, so that ``_native.host()`` can refuse the pair."""
    from unirl_amd import _native as N

    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler on this host")
    stub = "".join(f"int {name}(void) {{ return 4711; }}\n" for name in N.EXPORTED_SYMBOLS)
    (tmp_path / "stub.c").write_text(stub)
    subprocess.run([cc, "-shared", "-fPIC", "-o", str(tmp_path / "libunirl_hip.so"), str(tmp_path / "stub.c")], check=True)
    shutil.copy(N.HOST_PATH, tmp_path / N.HOST_PATH.name)
    code = ("import torch, importlib.util as u\n"
            f"s = u.spec_from_file_location('_unirl_torch_host', r'{tmp_path / N.HOST_PATH.name}')\n"
            "m = u.module_from_spec(s); s.loader.exec_module(m); print(m.abi_version)")
    out = subprocess.run([sys.executable, "-c", code], check=True, capture_output=True, text=True).stdout
    header = re.search(r"#define UNIRL_ABI_VERSION (\d+)", (ROOT / "include" / "unirl_hip.h").read_text()).group(1)
    assert out.split()[-1] == header == str(N.ABI_VERSION)

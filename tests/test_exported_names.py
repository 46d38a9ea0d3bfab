"""What the library exports to a host that links it: C names of its own prefix only (a host's function of the same name would be called in their place)."""
import shutil
import subprocess

import pytest


@pytest.fixture(scope="module")
def names():
    from qwengine_b200 import build, library_path
    build.build()
    nm = shutil.which("nm")
    if nm is None:
        pytest.skip("no nm")
    out = subprocess.run([nm, "-D", "--defined-only", library_path()], capture_output=True, text=True, check=True).stdout
    return [line.split()[-1] for line in out.splitlines() if line.strip()]


def test_c_names_carry_the_prefix(names):
    own = {n for n in names if n.startswith("q38b_")}
    assert "q38b_gemm_mx4" in own
    c_names = [n for n in names if n not in own and not n.startswith(("_Z", "_init", "_fini"))]
    assert c_names == []

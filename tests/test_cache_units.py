"""How the attention over a paged cache finds its work, replayed on the host
through the functions the kernels call (htree_amd/csrc/htree_cache_index.h,
tests/cache_units_check.cpp): every unit taken once, every slot inside the
workspace, the join reads the slots that the units of its rows wrote."""
import os
import shutil
import subprocess
import tempfile

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_unit_once():
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    with tempfile.TemporaryDirectory() as d:
        exe = os.path.join(d, "cache_units_check")
        subprocess.run([hipcc, "-x", "hip", "--offload-arch=gfx950", "-O2", "-std=c++17",
                        f"-I{ROOT}/include", f"-I{ROOT}/htree_amd/csrc",
                        os.path.join(ROOT, "tests", "cache_units_check.cpp"), "-o", exe],
                       check=True, capture_output=True)
        r = subprocess.run([exe], capture_output=True, text=True, timeout=600)
    print(r.stdout)
    assert r.returncode == 0, r.stdout
    assert " 0 failures" in r.stdout
    words = r.stdout.split()
    assert int(words[2]) > 100000 and int(words[4]) > 100000  # units, rows joined

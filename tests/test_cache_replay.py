"""The paged cache's index arithmetic replayed on the host through the
functions the kernels call (htree_amd/csrc/htree_cache_index.h,
tests/cache_replay_check.cpp), over ordinary and damaged lengths, tables and
trees: nothing out of bounds, every tile taken once, every walk ends."""
import os
import shutil
import subprocess
import tempfile

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_cache_indexes_in_bounds():
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    with tempfile.TemporaryDirectory() as d:
        exe = os.path.join(d, "cache_replay_check")
        subprocess.run([hipcc, "-x", "hip", "--offload-arch=gfx950", "-O2", "-std=c++17",
                        f"-I{ROOT}/include", f"-I{ROOT}/htree_amd/csrc",
                        os.path.join(ROOT, "tests", "cache_replay_check.cpp"), "-o", exe],
                       check=True, capture_output=True)
        r = subprocess.run([exe], capture_output=True, text=True, timeout=600)
    print(r.stdout)
    assert r.returncode == 0, r.stdout
    assert " 0 failures" in r.stdout
    assert int(r.stdout.split()[2]) > 10000  # units

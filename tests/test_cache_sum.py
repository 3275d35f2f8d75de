"""The sum that sizes the chunks of the attention over a paged cache, replayed
on the host through the functions the kernels call
(htree_amd/csrc/htree_cache_index.h, tests/cache_sum_check.cpp): the exact sum is
never above what the workspace holds, up to the most requests of a
call; more are refused (each block sums all lengths)."""
import ctypes
import os
import shutil
import subprocess
import tempfile

import pytest

from htree_amd import _native as N

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_chunks_cover_the_exact_sum():
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    with tempfile.TemporaryDirectory() as d:
        exe = os.path.join(d, "cache_sum_check")
        subprocess.run([hipcc, "-x", "hip", "--offload-arch=gfx950", "-O2", "-std=c++17",
                        f"-I{ROOT}/include", f"-I{ROOT}/htree_amd/csrc",
                        os.path.join(ROOT, "tests", "cache_sum_check.cpp"), "-o", exe],
                       check=True, capture_output=True)
        r = subprocess.run([exe], capture_output=True, text=True, timeout=600)
    print(r.stdout)
    assert r.returncode == 0, r.stdout
    assert " 0 failures" in r.stdout


def test_more_requests_are_refused():
    c = N.HtreeCache(1, 2, 128, 128, 16, 8, 16 * 256, 256, 128, 16 * 256, 256, 128)
    fake = ctypes.c_void_p(4096)  # never read: the calls are refused or empty
    n = ctypes.c_int64()
    for B, code in ((4096, N.HTREE_OK), (4097, N.HTREE_EUNSUPPORTED), (1 << 23, N.HTREE_EUNSUPPORTED)):
        assert N.lib().htree_draft_attention_workspace_bytes(c, B, 0, 32, 100, n) == code
        assert N.lib().htree_draft_attention(c, B, 0, 32, 100, 100, 1.0, fake, 4096, 128, fake, fake, fake, fake,
                                             fake, None, fake, 4096, 128, fake, 1 << 40, None) == code

"""Layers of a cache that share memory are refused by what moves tokens in
them, and no others: the check against the bytes themselves
(tests/layers_check.cpp, htree_amd/csrc/htree_layers.h), and the C entries'
refusals.  No launches."""
import ctypes
import os
import shutil
import subprocess
import tempfile

import pytest

from htree_amd import _native as N
from tests.test_cache_api import cache
from tests.test_step_api import at, copy, keep, pointers

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MIB = 1 << 20


def test_against_the_bytes():
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    with tempfile.TemporaryDirectory() as d:
        exe = os.path.join(d, "layers_check")
        subprocess.run([hipcc, "-x", "hip", "--offload-arch=gfx950", "-O2", "-std=c++17",
                        f"-I{ROOT}/include", f"-I{ROOT}/htree_amd/csrc",
                        os.path.join(ROOT, "tests", "layers_check.cpp"), "-o", exe],
                       check=True, capture_output=True)
        r = subprocess.run([exe], capture_output=True, text=True, timeout=600)
    print(r.stdout)
    assert r.returncode == 0, r.stdout
    words = r.stdout.replace(",", "").split()
    calls, shared = int(words[0]), int(words[2])
    assert shared > calls // 10 and calls - shared > calls // 10


def layers(*places):
    return (ctypes.c_void_p * len(places))(*places)


@pytest.mark.parametrize("f", [keep, copy])
def test_layers_that_share_memory_are_refused(f):
    """(Calls that are not refused would launch: those are tested on the GPU.)"""
    step = 8 * 16 * 256 * 2  # bytes of a layer's keys: eight pages of 16 tokens of 2 x 128 16-bit entries
    apart = dict(k=layers(8 * MIB, 9 * MIB), v=layers(10 * MIB, 11 * MIB))
    bad = [dict(v=apart["k"]),                                                # values are the keys
           dict(k=layers(8 * MIB, 8 * MIB)),                                  # a layer twice
           dict(k=layers(8 * MIB, 8 * MIB + step - 16)),                      # the last piece of a layer
           dict(v=layers(9 * MIB + step - 16, 11 * MIB)),                     # .. of keys, the first of values
           dict(k=layers(11 * MIB + 16, 9 * MIB)),
           dict(c=cache(k_page=0)), dict(c=cache(v_token=0)), dict(c=cache(k_head=0)), dict(c=cache(v_page=16 * 256 - 8)),
           dict(c=cache(k_head=64)), dict(c=cache(k_token=128))]
    bad += [dict([(name, at(9))]) for name in (("slots", "starts", "path", "kept") if f is keep else ("frm", "to", "tokens"))]
    for kw in bad:
        assert f(**{**apart, **kw}) == N.HTREE_EOVERLAP, kw
    assert f(**{**apart, "c": cache(k_page=1 << 56)}) == N.HTREE_EUNSUPPORTED
    # more layers than a few, one of them again as the last one's values
    many = [8 * MIB + 2 * i * step + (i == 5) * 1024 for i in range(300)]
    other = [8 * MIB + (2 * i + 1) * step + (i == 5) * 1024 for i in range(299)] + [many[17]]
    assert f(**{**apart, "layers": 300, "k": layers(*many), "v": layers(*other)}) == N.HTREE_EOVERLAP

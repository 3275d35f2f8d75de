"""The scale of draft_attention is taken in fp32, times log2(e): what is not a
finite number there is refused, at the C entry and in Python."""
import ctypes
import math

import pytest
import torch

import htree_amd
from htree_amd import _native as N

FAKE = ctypes.c_void_p(4096)  # never read: the calls are refused or empty
BAD = [math.nan, math.inf, -math.inf, 1e39, -1e300, 2.4e38, -2.4e38]


def call(scale):
    c = N.HtreeCache(1, 2, 128, 128, 16, 8, 16 * 256, 256, 128, 16 * 256, 256, 128)
    return N.lib().htree_draft_attention(c, 4, 0, 32, 100, 100, scale, FAKE, 4096, 128, FAKE, FAKE, FAKE, FAKE, FAKE,
                                         None, FAKE, 4096, 128, FAKE, 1 << 40, None)


@pytest.mark.parametrize("scale", BAD)
def test_the_c_entry_refuses(scale):
    assert call(scale) == N.HTREE_ESHAPE


@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-45, -1.0, 2.35e38, -2.35e38])
def test_the_c_entry_takes(scale):
    assert call(scale) == N.HTREE_OK


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 0])
def test_python(rows):
    f = lambda *n: torch.zeros(n, dtype=torch.bfloat16, device="cuda:0")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda:0")
    args = [f(rows, 8, 64), f(4, 16, 2, 64), f(4, 16, 2, 64), i32([[0, 1, 2]]), i32([40]), i32([0, rows])]
    for scale in BAD:
        with pytest.raises(AssertionError):
            htree_amd.draft_attention(*args, scale=scale)
            print("not refused:", scale, flush=True)
    assert htree_amd.draft_attention(*args, scale=2.35e38).shape == (rows, 8, 64)

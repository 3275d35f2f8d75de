"""GPU tests of draft_attention over batches as large as a call takes."""
import numpy as np
import pytest
import torch

import htree_amd
from htree_amd.cache import MAX_REQUESTS
from tests.test_gpu_draft import Case, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B", [65, 1000, MAX_REQUESTS])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_large_batches(B, dtype):
    """Short requests, none at all among them, and a few long enough to be
    split, the last one too."""
    g = np.random.default_rng(B)
    lens = g.integers(0, 40, B)
    lens[[B // 3, B // 2, B - 1]] = 3000, 700, 1500
    new = np.minimum(lens, g.integers(0, 3, B))
    c = Case(lens.tolist(), new.tolist(), 4, 2, 32, 32, dtype, seed=B, width=200)
    c.check(c.run())


def test_more_requests_are_refused():
    B = MAX_REQUESTS + 1
    q = torch.zeros(4, 4, 32, device="cuda:0")
    k = torch.zeros(3, 16, 2, 32, device="cuda:0")
    with pytest.raises(AssertionError, match="at most"):
        htree_amd.draft_attention(q, k, k, i32(np.zeros((B, 2))), i32(np.ones(B)), i32(np.zeros(B + 1)))

"""GPU tests of head_norm at the most rows and heads of a call, for heads that
are read in 8-byte pieces and take twice the lanes."""
import pytest
import torch

import htree_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype,D,lanes", [(torch.float32, 252, 64), (torch.bfloat16, 248, 32)])
def test_most_heads_of_narrow_pieces(dtype, D, lanes):
    """Rows that are one row, so that every output is the first one's; one more
    row is refused."""
    heads, kv = 30, 2
    rows = (1 << 32) // lanes // (heads + kv)
    g = torch.Generator(device=DEV).manual_seed(D)
    q, k = (torch.randn(1, h, D, generator=g, device=DEV).to(dtype) for h in (heads, kv))
    w = torch.randn(D, generator=g, device=DEV)
    want = htree_amd.head_norm(q, k, w, w)
    wide = lambda x, n: x.expand(n, *x.shape[1:])
    with pytest.raises(AssertionError):
        htree_amd.head_norm(wide(q, rows), wide(k, rows), w, w)
    for got, one in zip(htree_amd.head_norm(wide(q, rows - 1), wide(k, rows - 1), w, w), want):
        assert all(bool((x == one).all()) for x in got.split(1 << 18))

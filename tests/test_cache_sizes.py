"""Sizes past the 32 bits that the C ABI takes are refused: wrapped, they were
other calls (2^32 + 5 pages were 5)."""
import pytest
import torch

import htree_amd
from htree_amd import cache

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PAST = [2 ** 31, 2 ** 32, 2 ** 32 + 5]


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("n", PAST)
def test_page_tables(n):
    args = dict(ctx_lens=i32([1]), new_lens=i32([1]), block_table=i32([[0, -1]]), free_pages=i32([1]), page_size=16,
                num_pages=5, rows=1)
    htree_amd.page_tables(**args)
    for name in ("num_pages", "rows"):
        with pytest.raises(AssertionError, match="31 bits"):
            htree_amd.page_tables(**dict(args, **{name: n}))
    with pytest.raises(AssertionError):
        htree_amd.page_tables(**dict(args, page_size=n))


@pytest.mark.parametrize("n", PAST)
def test_expanded_tensors(n):
    """Views of a few bytes with that many rows, heads or pages."""
    f = lambda *s: torch.zeros(s, device=DEV)
    kc = f(3, 16, 1, 32)
    many = lambda x, dim: x.expand(*(n if i == dim else s for i, s in enumerate(x.shape)))
    call = lambda q, k: htree_amd.draft_attention(q, k, k, i32([[0, 1]]), i32([20]), i32([0, 1]))
    call(f(1, 1, 32), kc)
    for q in (many(f(1, 1, 32), 0), many(f(1, 1, 32), 1)):
        with pytest.raises(AssertionError, match="below 2"):
            call(q, kc)
    with pytest.raises(AssertionError, match="less than 2"):
        call(f(1, 1, 32), many(f(1, 16, 1, 32), 0))
    slots = torch.zeros(1, dtype=torch.int64, device=DEV)
    with pytest.raises(AssertionError, match="below 2"):
        htree_amd.cache_append(many(f(1, 1, 32), 0), many(f(1, 1, 32), 0), kc, kc.clone(), slots.expand(n))
    with pytest.raises(AssertionError, match="q must be"):
        htree_amd.cache_append(f(1, 1, 32), f(1, 1, 32), kc, kc.clone(), slots, q=many(f(1, 1, 32), 1),
                               positions=i32([0]), cos=f(4, 16), sin=f(4, 16))
    with pytest.raises(AssertionError, match="cos and sin"):
        htree_amd.cache_append(f(1, 1, 32), f(1, 1, 32), kc, kc.clone(), slots, positions=i32([0]),
                               cos=many(f(1, 16), 0), sin=many(f(1, 16), 0))
    assert cache.INT32 == 2 ** 31

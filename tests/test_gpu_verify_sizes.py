"""GPU tests of verify_drafts at the most rows that a call takes: what it
writes of the path ends with the path."""
import pytest
import torch

import htree_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROWS, GUARD = 2 ** 31 - 1, 1 << 16


@pytest.mark.parametrize("greedy", [True, False])
def test_most_rows(greedy):
    """Requests at both ends of 2^31 - 1 rows, one token in the vocabulary, which
    every draft is and the target always says."""
    buf = torch.empty(ROWS + 2 * GUARD, dtype=torch.int32, device=DEV)
    out = htree_amd.Verified(torch.empty(2, dtype=torch.int32, device=DEV), buf[GUARD:-GUARD],
                             torch.empty(2, dtype=torch.int64, device=DEV))
    p = torch.ones(1, 1, device=DEV).expand(ROWS, 1)
    tokens = torch.zeros(ROWS, dtype=torch.int64, device=DEV)
    numbers = () if greedy else (torch.zeros(ROWS, device=DEV), torch.zeros(2, device=DEV))
    for starts, new in (([0, 2, 3], [2, 1]), ([ROWS - 5, ROWS - 3, ROWS], [2, 3]), ([ROWS - 1, ROWS, ROWS], [1, 0])):
        buf.fill_(-9)
        htree_amd.verify_drafts(p, tokens, torch.tensor(starts, dtype=torch.int32, device=DEV), *numbers, out=out)
        assert out.kept.tolist() == new and out.next_tokens.tolist() == [0 if n else -1 for n in new]
        for s, n in zip(starts, new):
            assert out.path[s:s + n].tolist() == list(range(n))
            out.path[s:s + n] = -1
        assert bool((out.path == -1).all())
        assert bool((buf[:GUARD] == -9).all()) and bool((buf[-GUARD:] == -9).all())

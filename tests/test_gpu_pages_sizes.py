"""GPU tests of fork_requests and unused_pages at the widest block table that
a call takes."""
import pytest
import torch

import htree_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
WIDTH, GUARD = 2 ** 31 - 1, 1 << 16


def test_widest_table():
    """A row of 2^31 - 1 entries: a forked one ends where it ends, and its last
    entries are read too."""
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    table = torch.full((1, WIDTH), -1, dtype=torch.int32, device=DEV)
    table[0, :3] = i32([4, 2, 7])
    table[0, -2:] = i32([5, 1])
    buf = torch.full((WIDTH + 2 * GUARD,), -9, dtype=torch.int32, device=DEV)
    out = htree_amd.Forked(buf[GUARD:-GUARD].view(1, WIDTH), *(i32([-9]) for _ in range(5)))
    for page, length, live in ((16, 33, 3), (1, WIDTH, WIDTH), (1, WIDTH - 1, WIDTH - 1)):
        buf.fill_(-9)
        htree_amd.fork_requests(table, i32([length]), i32([0]), i32([9]), page, 12, out=out)
        assert out.lens.tolist() == [length] and out.copy_from.tolist() == [-1] and out.pages_used.tolist() == [0]
        assert torch.equal(out.block_table[:, :live], table[:, :live])
        assert bool((out.block_table[:, live:] == -1).all())
        assert bool((buf[:GUARD] == -9).all()) and bool((buf[-GUARD:] == -9).all())
        u = htree_amd.unused_pages(table, i32([length]), page, 12)
        used = {4, 2, 7} | ({5} if live > 3 else set()) | ({1} if live == WIDTH else set())
        want = [p for p in range(12) if p not in used]
        assert int(u.count) == len(want) and u.pages.tolist() == want + [-1] * len(used)

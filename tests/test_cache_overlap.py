"""page_tables writes the block table while other blocks read the lengths, the
parents and the page list: a table that overlaps one of them is refused."""
import pytest
import torch

import htree_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def args():
    """Two requests, every tensor in a buffer of its own."""
    new = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)
    return dict(ctx_lens=new(2), new_lens=new(2) + 1, block_table=new(2, 4), free_pages=new(5), page_size=16,
                num_pages=9, rows=3, parents=new(3) - 1)


@pytest.mark.parametrize("name", ["ctx_lens", "new_lens", "free_pages", "parents"])
@pytest.mark.parametrize("at", [0, 3, 7])
def test_a_table_over_an_input(name, at):
    a = args()
    buf = torch.zeros(40, dtype=torch.int32, device=DEV)
    a["block_table"] = buf[:8].view(2, 4)
    a[name] = buf[at:at + a[name].numel()]
    with pytest.raises(AssertionError, match="block_table"):
        htree_amd.page_tables(**a)
    a[name] = buf[8:8 + a[name].numel()]  # right behind it: taken
    htree_amd.page_tables(**a)
    a["block_table"] = buf[8 + a[name].numel():][:8].view(2, 4)  # and right before it
    htree_amd.page_tables(**a)
    torch.cuda.synchronize()


def test_inputs_may_share_memory():
    """Tensors that are only read may be the same."""
    a = args()
    a["new_lens"] = a["ctx_lens"]
    t = htree_amd.page_tables(**a)
    assert t.lens.tolist() == [0, 0]

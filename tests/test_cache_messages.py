"""What the serving calls say of what they refuse."""
import pytest
import torch

from htree_amd import _native as N
from htree_amd.cache import check_table


@pytest.mark.parametrize("rc", [N.HTREE_ESHAPE, N.HTREE_EUNSUPPORTED])
def test_statuses_name_the_serving_limits(rc):
    assert "serving" in N.strerror(rc)
    assert "htree_tree" not in N.strerror(N.HTREE_EWORKSPACE)


def test_expanded_tables_are_refused_as_such():
    t = torch.zeros(1, 4, dtype=torch.int32)
    check_table(t, 1, t.device)
    check_table(torch.zeros(3, 8, dtype=torch.int32)[:, :4], 3, t.device)
    with pytest.raises(AssertionError, match="expanded"):
        check_table(t.expand(3, 4), 3, t.device)
    check_table(t[:, :0].expand(3, 0), 3, t.device)  # no entries

"""The most rows and heads that head_norm takes: 2^32 threads, of which a head
has as many as its pieces, 16 bytes of each half or, where a half is no whole
ones, 8.  No launches."""
import pytest

from htree_amd import _native as N
from tests.test_step_api import norm


def lanes(D, size):
    """A head's, from its sizes alone."""
    half = D * size // 2
    pieces = half // 16 if half % 16 == 0 else half // 8
    return 1 << (pieces - 1).bit_length()


@pytest.mark.parametrize("dtype,D,of_a_head", [(0, 256, 32), (0, 252, 64), (0, 132, 64), (0, 124, 32), (0, 4, 1), (1, 256, 16),
                                               (1, 248, 32), (1, 24, 4), (2, 24, 4), (1, 8, 1)])
def test_more_threads_than_a_grid(dtype, D, of_a_head):
    size = 4 if dtype == 0 else 2
    assert lanes(D, size) == of_a_head
    assert of_a_head >= (D / 4 if D * size % 32 else D / 8) / (1 if dtype == 0 else 2)  # as the documentation has it
    heads = 32
    for more in (0, 1):  # rows x heads at the limit, and behind it
        rows = min((1 << 32) // of_a_head // heads + more, (1 << 31) // heads)
        assert norm(dtype=dtype, rows=rows, H=heads - 2, Hkv=2, D=D, qr=D * heads) == N.HTREE_EUNSUPPORTED

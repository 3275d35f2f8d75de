"""GPU tests of keep_drafts and copy_pages where blocks take several layers
(kept drafts of many requests and layers) and where a page's tokens are more
than its blocks read at once."""
import numpy as np
import pytest
import torch

import htree_amd
from tests.test_gpu_pages import DEV, caches, i32, moved, steps

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout,layers,H,K,V,dtype", [
    ("stacked", 70, 1, 8, 8, "float16"), ("list", 129, 1, 4, 8, "float32"), ("stacked", 27, 16, 128, 128, "bfloat16"),
    ("heads first", 33, 2, 96, 96, "bfloat16"), ("beside", 66, 5, 8, 16, "bfloat16"), ("list", 64, 2, 64, 32, "float16")])
def test_several_layers_a_block(layout, layers, H, K, V, dtype):
    """More than 1024 blocks of one layer, and last blocks of one to four layers."""
    B = 40
    slots, starts, path, kept, pages = steps(B, 19, 16, np.random.default_rng(layers))
    k, v, ks, vs = caches(layout, layers, pages, 16, H, K, V, dtype, 3)
    pieces = H * (K + V) * ks[0].element_size() // 16
    assert B * layers * -(-pieces // 256) > 1024  # (from here on four layers a block)
    pairs = [(slots[starts[b] + path[starts[b] + j]], slots[starts[b] + j]) for b in range(B) for j in range(kept[b])]
    want = [moved(x, pairs, 16) for x in ks + vs]
    htree_amd.keep_drafts(k, v, torch.as_tensor(slots).to(DEV), i32(starts), i32(path), i32(kept))
    for x, y in zip(ks + vs, want):
        assert torch.equal(x, y)


@pytest.mark.parametrize("page,H,D,dtype", [(256, 16, 128, "bfloat16"), (4096, 16, 128, "float16"), (1024, 9, 256, "float32"),
                                            (4096, 1, 8, "bfloat16"), (512, 3, 40, "bfloat16")])
@pytest.mark.parametrize("whole", [False, True])
def test_large_pages(page, H, D, dtype, whole):
    g = np.random.default_rng(page + D)
    pages, n = 13, 6
    perm = g.permutation(pages)
    frm, to, count = perm[:n].copy(), perm[n:2 * n].copy(), g.integers(1, page, n)
    count[:4] = [page, page - 1, 65, 1]
    frm[5] = frm[0]
    k, v, ks, vs = caches("stacked", 2, pages, page, H, D, D, dtype, 4)
    want = []
    for x in ks + vs:
        y = x.clone()
        for a, b, c in zip(frm, to, count):
            y[b, :page if whole else c] = x[a, :page if whole else c]
        want.append(y)
    htree_amd.copy_pages(k, v, i32(frm), i32(to), None if whole else i32(count))
    for x, y in zip(ks + vs, want):
        assert torch.equal(x, y)

"""GPU tests of keep_drafts and copy_pages on caches that share a buffer:
layers, keys and values between each other in any order are moved, what shares
an entry is refused and left as it is."""
import numpy as np
import pytest
import torch

import htree_amd
from tests.test_gpu_pages import DEV, i32, moved, steps

pytestmark = pytest.mark.gpu
PAGE, H, K = 16, 2, 32


def shared_buffer(kind, layers, pages):
    """Layers' keys and values in one buffer."""
    g = torch.Generator(device=DEV).manual_seed(layers)
    rand = lambda *n: torch.randn(*n, generator=g, device=DEV).bfloat16()
    if kind == "layer, keys and values":
        x = rand(layers, 2, pages, PAGE, H, K)
        return x[:, 0], x[:, 1]
    if kind == "inside pages":
        x = rand(pages, layers, 2, H, PAGE, K).permute(1, 2, 0, 4, 3, 5)
        return x[:, 0], x[:, 1]
    if kind == "some layers, the last first":
        x = rand(pages, PAGE, H, 3 * layers, 2 * K)
        order = [3 * l + (l % 3 == 1) for l in reversed(range(layers))]
        return [x[:, :, :, l, :K] for l in order], [x[:, :, :, l, K:] for l in order]
    assert kind == "keys of one layer with values of another"
    x = rand(layers + 1, pages, PAGE, 2, H, K)
    return [x[l, :, :, 0] for l in range(layers)], [x[l + 1, :, :, 1] for l in range(layers)]


@pytest.mark.parametrize("layers", [1, 5, 70])
@pytest.mark.parametrize("kind", ["layer, keys and values", "inside pages", "some layers, the last first",
                                  "keys of one layer with values of another"])
def test_layers_in_one_buffer(kind, layers):
    slots, starts, path, kept, pages = steps(5, 20, PAGE, np.random.default_rng(layers))
    k, v = shared_buffer(kind, layers, pages)
    pairs = [(slots[starts[b] + path[starts[b] + j]], slots[starts[b] + j]) for b in range(5) for j in range(kept[b])]
    want = [moved(x, pairs, PAGE) for x in [*k, *v]]
    htree_amd.keep_drafts(k, v, torch.as_tensor(slots).to(DEV), i32(starts), i32(path), i32(kept))
    assert all(torch.equal(x, y) for x, y in zip([*k, *v], want))
    want = [moved(x, [(t, 2 * PAGE + t) for t in range(PAGE)], PAGE) for x in want]
    htree_amd.copy_pages(k, v, i32([0]), i32([2]))
    assert all(torch.equal(x, y) for x, y in zip([*k, *v], want))


def test_shared_entries_are_refused():
    x = torch.randn(9, 4, PAGE, H, K, device=DEV)
    before = x.clone()
    ints = torch.zeros(4 * PAGE * H * K, dtype=torch.int32, device=DEV)
    slots, lists = torch.arange(4, device=DEV), (i32([0, 4]), i32([0, 2, 3, -1]), i32([3]))
    keep = lambda k, v, s=slots, l=lists: htree_amd.keep_drafts(k, v, s, *l)
    copy = lambda k, v, a=i32([0]), b=i32([1]), n=i32([5]): htree_amd.copy_pages(k, v, a, b, n)
    flat = x.view(-1)
    inside = ints.view(torch.float32).view(4, PAGE, H, K)
    bad = []
    for f in (keep, copy):
        bad += [lambda f=f: f(x[0:4], x[2:6]), lambda f=f: f(x[0:4], x[3:7]), lambda f=f: f([x[0], x[1]], [x[2], x[1]]),
                lambda f=f: f(x[0], flat[4:4 + x[0].numel()].view(x[0].shape)),
                lambda f=f: f(flat.as_strided((3, 4, PAGE, H, K), (x.stride(1), *x.stride()[1:])), x[7]),
                lambda f=f: f(flat.as_strided((4, PAGE, H, K), (H * K * 8, H * K, K, 1)), x[7]),
                lambda f=f: f(flat.as_strided((4, PAGE, H, K), (PAGE * H * K, H * K, 4, 1)), x[7]),
                lambda f=f: f(x[..., :24], x[..., 16:])]
    bad += [lambda: keep(inside, x[0], l=(ints[:2], *lists[1:])), lambda: keep(x[0], inside, l=(lists[0], ints[4:8], lists[2])),
            lambda: keep(inside, x[0], l=(*lists[:2], ints[-1:])), lambda: copy(inside, x[0], a=ints[:1]),
            lambda: copy(inside, x[0], b=ints[-1:]), lambda: copy(x[0], inside, n=ints[77:78])]
    for i, call in enumerate(bad):
        with pytest.raises(AssertionError):
            call()
            print("not refused:", i)
    assert torch.equal(x, before) and not ints.any()
    keep(x[..., :16], x[..., 16:]), copy(x[0:3], x[3:6])  # beside each other

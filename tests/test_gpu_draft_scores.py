"""GPU tests of draft_attention where the scores are so large that only a row's
highest ones count: scales up to 2^100, keys and queries of small whole numbers,
so that every score is exact and the output is the mean of the values of the
tokens with the highest."""
import numpy as np
import pytest
import torch

import htree_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def cached(x):
    """x [L, H_kv, D] in pages of 16, in order."""
    pages = -(-x.shape[0] // 16)
    c = torch.zeros(pages * 16, *x.shape[1:], dtype=x.dtype)
    c[:x.shape[0]] = x
    return c.view(pages, 16, *x.shape[1:]).to(DEV)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# few rows and many, split over their tokens or not, one wave's tokens alone
SIZES = [(9, 1), (1000, 1), (1010, 40), (4100, 1), (5000, 24), (2000, 300)]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("L,new", SIZES)
@pytest.mark.parametrize("scale", [2.0 ** e for e in (8, 13, 14, 16, 20, 24, 26, 40, 100)] + [-2.0 ** 15, -2.0 ** 60])
@pytest.mark.parametrize("shift", [0, -40])
def test_the_highest_scores_alone(dtype, L, new, scale, shift):
    """Scores are whole numbers times `scale`, 256 at least: a token a step
    below the highest weighs e^-256 of it, which is zero in the result.

    What is left: the values' sum over n tokens of equal weight (each sum in
    fp32, n + 4 steps of 2^-24 of the mean |v|, twice with the weights' own),
    their common weight cancels, and the result's half step."""
    H, Hkv, D = 4, 1, 64
    g = torch.Generator().manual_seed(L + new)
    t = DT[dtype]
    q = torch.randint(-2, 3, (new, H, D), generator=g).to(t)
    k = torch.randint(-2, 3, (L, Hkv, D), generator=g).to(t)
    q[..., 0] = 1
    k[..., 0] = shift          # all of a row's scores below 0, or about it
    v = torch.randn(L, Hkv, D, generator=g).to(t)
    out = htree_amd.draft_attention(q.to(DEV), cached(k), cached(v), i32([list(range(-(-L // 16)))]), i32([L]),
                                    i32([0, new]), scale=scale)
    torch.cuda.synchronize()
    got = out.double().cpu().numpy()
    s = np.einsum("nhd,ld->nhl", q.double().numpy(), k.double().numpy()[:, 0]) * np.sign(scale)
    see = np.arange(L)[None] <= (L - new + np.arange(new))[:, None]
    s = np.where(see[:, None], s, -np.inf)
    w = (s == s.max(-1, keepdims=True)).astype(np.float64)
    n = w.sum(-1, keepdims=True)
    vv = v.double().numpy()[:, 0]
    want, A = w @ vv / n, w @ np.abs(vv) / n
    fi = torch.finfo(t)
    b = A * 2 * (n + 4) * 2.0 ** -24
    bar = b + (np.abs(want) + b) * (fi.eps / 2) + fi.tiny * fi.eps
    err = np.abs(got - want)
    bad = ~(err <= bar)
    assert not bad.any(), f"{int(bad.sum())} of {bad.size}: {got[bad][0]} for {want[bad][0]} (bar {bar[bad][0]})"


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("new", [1, 40])
def test_scores_that_cross_from_far_below_to_far_above(dtype, new):
    """The highest score rises from tile to tile, from -2^30 to 2^30 log2
    units and through zero; a drafted branch that sees none of the last ones
    keeps to its own."""
    L, H, D = 900, 2, 32
    t = DT[dtype]
    g = torch.Generator().manual_seed(3)
    q = torch.ones(new, H, D).to(t)
    q[..., 1:] = 0
    k = torch.zeros(L, 1, D).to(t)
    step = torch.arange(L) - 400
    k[:, 0, 0] = step.float().clamp(-256, 256).to(t)  # whole numbers that every type holds
    v = torch.randn(L, 1, D, generator=g).to(t)
    scale = 2.0 ** 21.5
    parents = torch.full((new,), -1, dtype=torch.int32)  # siblings: each sees the cached tokens and itself
    keys = k[:, 0, 0].double().numpy()
    out = htree_amd.draft_attention(q.to(DEV), cached(k), cached(v), i32([list(range(-(-L // 16)))]), i32([L]),
                                    i32([0, new]), parents=parents.to(DEV), scale=scale)
    torch.cuda.synchronize()
    got, vv = out.double().cpu().numpy(), v.double().numpy()[:, 0]
    fi = torch.finfo(t)
    for j in range(new):
        see = np.arange(L) < L - new
        see[L - new + j] = True
        w = see & (keys == keys[see].max())
        n = w.sum()
        want, A = w @ vv / n, w @ np.abs(vv) / n
        b = A * 2 * (n + 4) * 2.0 ** -24
        bar = b + (np.abs(want) + b) * (fi.eps / 2) + fi.tiny * fi.eps
        assert np.all(np.abs(got[j] - want[None]) <= bar[None]), j


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("new", [5, 40])
def test_infinities_beside_large_scores(dtype, new):
    """A drafted token with an infinite value reaches the rows that see it,
    in that dim alone, where its score is the highest of large ones."""
    L, H, D = 300, 4, 64
    t = DT[dtype]
    g = torch.Generator().manual_seed(4)
    q, k = torch.zeros(new, H, D), torch.zeros(L, 1, D)
    q[..., 0], k[..., 0] = 1, torch.randint(-3, 4, (L, 1), generator=g).float()
    at = L - new + 2
    k[at, :, 0] = 4
    v = torch.randn(L, 1, D, generator=g)
    q, k, v = q.to(t), k.to(t), v.to(t)
    vc = cached(v)
    vc[at // 16, at % 16, 0, 7] = float("inf")
    parents = torch.full((new,), -1, dtype=torch.int32)
    parents[3] = 2
    out = htree_amd.draft_attention(q.to(DEV), cached(k), vc, i32([list(range(-(-L // 16)))]), i32([L]),
                                    i32([0, new]), parents=parents.to(DEV), scale=2.0 ** 40)
    torch.cuda.synchronize()
    got, vv = out.double().cpu().numpy(), v.double().numpy()[:, 0]
    keys = k[:, 0, 0].numpy(force=True) if t is not torch.bfloat16 else k[:, 0, 0].float().numpy()
    fi = torch.finfo(t)
    for j in range(new):
        see = np.arange(L) < L - new
        see[L - new + j] = True
        if j == 3:
            see[at] = True
        w = see & (keys == keys[see].max())
        n = w.sum()
        want, A = w @ vv / n, w @ np.abs(vv) / n
        b = A * 2 * (n + 4) * 2.0 ** -24
        bar = b + (np.abs(want) + b) * (fi.eps / 2) + fi.tiny * fi.eps
        dims = np.arange(D) != 7 if j in (2, 3) else np.ones(D, bool)
        assert np.all(np.abs(got[j] - want[None])[:, dims] <= bar[None, dims]), j
        assert np.isposinf(got[j][:, ~dims]).all()

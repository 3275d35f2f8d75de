"""GPU tests of draft_attention where most of a row's weights are tiny: one
token with a far larger score and values of zero, a long flat tail behind it
that the output comes from alone; and scores that rise from token to token, so
that the maximum moves again and again."""
import numpy as np
import pytest
import torch

import htree_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def attend(q, k, v, width=None, parents=None):
    """One request: all of q's rows are its last tokens.  Pages of 16, in the
    cache's order; `width`: of the table."""
    L, Hkv, K = k.shape
    pages = -(-L // 16)
    cache = []
    for x in (k, v):
        c = torch.zeros(pages * 16, Hkv, x.shape[2], dtype=x.dtype)
        c[:L] = x
        cache.append(c.view(pages, 16, Hkv, x.shape[2]).to(DEV))
    table = torch.full((1, max(width or pages, pages)), -1, dtype=torch.int32)
    table[0, :pages] = torch.arange(pages, dtype=torch.int32)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    out = htree_amd.draft_attention(q.to(DEV), *cache, table.to(DEV), i32([L]), i32([0, q.shape[0]]), parents=parents)
    torch.cuda.synchronize()
    return out.double().cpu().numpy()


def reference(q, k, v, dtype):
    """Output and error bound, in 64 bits.

    Scores: K products of |q||k| summed in fp32, scaled and times log2 e, each
    step off by 2^-24 of sum |q||k| scale at most, exp2 by 2^-22: e in the
    exponent, so 2 e of A = sum p |v| / sum p between numerator and sum.  Sums
    of L terms in any order: L 2^-24 each.  A 16-bit P is off by half a step,
    in the numerator and the sum alike: dp (v - o).  fp16's is off by 2^-36 of
    the largest weight where that is more: the largest weighs 2^11 in it at
    least, and its step is 2^-24 at least.  The result is off by half a step of
    the type, or half its smallest number."""
    n, H, K = q.shape
    L, Hkv, V = v.shape
    fi = torch.finfo(DT[dtype])
    half, u = fi.eps / 2, 2.0 ** -24
    q, k, v = (x.double().numpy() for x in (q, k, v))
    see = np.arange(L)[None] <= (L - n + np.arange(n))[:, None]
    out, bar = np.zeros((n, H, V)), np.zeros((n, H, V))
    for h in range(H):
        kk, vv, qq = k[:, h * Hkv // H], v[:, h * Hkv // H], q[:, h]
        s = np.where(see, qq @ kk.T * K ** -0.5, -np.inf)
        mag = np.where(see, np.abs(qq) @ np.abs(kk).T * K ** -0.5, 0).max(-1)
        p = np.exp(s - s.max(-1, keepdims=True))
        den = p.sum(-1, keepdims=True)
        o = p @ vv / den
        A = p @ np.abs(vv) / den
        e = ((K + 8) * u * mag + 2.0 ** -22)[:, None]
        b = A * (2 * e + (2 * L + 16) * u)
        if dtype != "float32":
            b = b + (A + np.abs(o)) * half
        if dtype == "float16":
            b = b + 2.0 ** -36 * (see @ np.abs(vv) + see.sum(-1, keepdims=True) * np.abs(o)) / den
        out[:, h], bar[:, h] = o, b * 1.001 + (np.abs(o) + b) * half + fi.tiny * fi.eps / 2
    return out, bar


def check(got, want, bar, what):
    err = np.abs(got - want)
    bad = ~(err <= bar)
    print(what, "worst", float((err / bar).max()), "relative", float((err / np.abs(want).max()).max()), flush=True)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.size}, {got[bad][0]} for {want[bad][0]} (bar {bar[bad][0]})"


# tokens, new ones: single tokens and few, split over the tokens or not (a
# table of at most 1024 tokens is not), and many rows in both ways
SIZES = [(1000, 1), (1010, 40), (4096, 1), (5000, 24), (1500, 1500), (33000, 3)]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("L,new", SIZES)
@pytest.mark.parametrize("gap", [12, 17, 20, 24])
def test_a_dominant_token_without_values(dtype, L, new, gap):
    """gap: log2 units that the tail's scores lie below the token's."""
    H, Hkv, D = (4, 1, 64) if new < 1000 else (2, 1, 32)
    g = torch.Generator().manual_seed(L + gap)
    t = DT[dtype]
    q = torch.randn(new, H, D, generator=g).to(t)
    k = (torch.randn(L, Hkv, D, generator=g) * 0.2).to(t)
    v = (32 + 16 * torch.rand(L, Hkv, D, generator=g)).to(t)
    q[..., 0] = 8
    k[..., 0] = 0
    at = 5
    k[at] = 0
    k[at, :, 0] = gap * np.log(2) * D ** 0.5 / 8
    v[at] = 0
    want, bar = reference(q, k, v, dtype)
    check(attend(q, k, v), want, bar, f"{dtype} L {L} new {new} gap {gap}")


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("L,new", SIZES[:4])
@pytest.mark.parametrize("rise", [0.01, 0.05, 0.4])
def test_scores_that_rise(dtype, L, new, rise):
    """Each token's score lies `rise` log2 units above the one before it, up
    to where the type's keys end."""
    H, Hkv, D = 4, 1, 64
    g = torch.Generator().manual_seed(L)
    t = DT[dtype]
    q = (torch.randn(new, H, D, generator=g) * 0.5).to(t)
    k = (torch.randn(L, Hkv, D, generator=g) * 0.2).to(t)
    v = torch.randn(L, Hkv, D, generator=g).to(t)
    q[..., 0] = 8
    k[:, 0, 0] = (torch.arange(L) * (rise * np.log(2) * D ** 0.5 / 8)).to(t)
    want, bar = reference(q, k, v, dtype)
    check(attend(q, k, v), want, bar, f"{dtype} L {L} new {new} rise {rise}")

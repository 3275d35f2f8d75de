"""GPU tests of draft_attention against the definition in 64 bits, with the
pool's other pages and the ends of partly filled ones full of NaN."""
import numpy as np
import pytest
import torch

import htree_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def i32(x):
    return torch.as_tensor(np.asarray(x, np.int64)).to(torch.int32).to(DEV)


def tree(kind, n, g):
    if kind == "chain":
        return np.arange(n) - 1
    if kind == "star":
        return np.full(n, -1)
    return np.array([max(-1, j - 1 - int(g.integers(0, 6))) for j in range(n)], np.int64)


def visible(kind, parents, n, ctx, length):
    """[n, length] what each new token sees."""
    see = np.zeros((n, length), bool)
    see[:, :max(ctx, 0)] = True
    for j in range(n):
        a = j
        while a >= 0:
            if 0 <= ctx + a < length:
                see[j, ctx + a] = True
            p = (a - 1) if kind is None else int(parents[a])
            a = p if 0 <= p < a else -1
    if kind is None:  # a chain over negative contexts: tokens before the row
        for j in range(n):
            see[j] = np.arange(length) <= ctx + j
    return see


def reference(q, k, v, see, scale, dtype):
    """Output and error bound of one request: q [n, H, K], k / v [L, H_kv, .]
    in float64, see [n, L].

    Scores: K products of at most |q||k| summed in fp32, then scaled: each of
    the K + 2 steps is off by 2^-24 of sum |q||k| scale at most; p = exp(s - m)
    to 2^-22 relative, and the log2 form's product with log2 e to 3 x 2^-24 of
    |s| + |m|.  With e the largest of these, numerator and denominator are off
    by e each, relative to A = sum p |v| / sum p.  Sums of L terms in fp32, in
    any order: L 2^-24 each.  16-bit types round P, in the numerator and in the
    sum alike: sum dp (v - o) / sum p is off by half a step of A + |o| at most;
    and the result (half a step of it)."""
    n, H, K = q.shape
    L, Hkv, V = v.shape
    out, bar = np.zeros((n, H, V)), np.zeros((n, H, V))
    if L == 0:
        return out, bar
    half = torch.finfo(DT[dtype]).eps / 2
    u = 2.0 ** -24
    tiny = torch.finfo(DT[dtype]).tiny
    for h in range(H):
        kk, vv, qq = k[:, h * Hkv // H], v[:, h * Hkv // H], q[:, h]
        s = np.where(see, qq @ kk.T * scale, -np.inf)
        mag = np.where(see, np.abs(qq) @ np.abs(kk).T * abs(scale), 0).max(-1)
        m = s.max(-1, initial=-np.inf)
        live = np.isfinite(m)
        p = np.where(see, np.exp(s - np.where(live, m, 0)[:, None]), 0)
        den = np.where(live, p.sum(-1), 1)
        o = p @ vv / den[:, None]
        A = p @ np.abs(vv) / den[:, None]
        e = (K + 2 + 6) * u * mag + 2.0 ** -22
        b = A * (2 * e + (2 * L + 16) * u)[:, None]
        if dtype != "float32":
            b = b + (A + np.abs(o)) * half
        out[:, h] = o
        bar[:, h] = b * 1.001 + (np.abs(o) + b) * (half if dtype != "float32" else 4 * u) + tiny
    return out, bar


class Case:
    """A batch over a pool of pages: lens, new tokens and trees per request."""

    def __init__(self, lens, new, H, Hkv, K, V, dtype, page=16, kind=None, seed=0, spare=5, pad=0,
                 heads_first=False, width=None, dev=DEV):
        g = np.random.default_rng(seed)
        tg = torch.Generator().manual_seed(seed)
        t = DT[dtype]
        self.lens, self.new, self.kind, self.dtype, self.page = list(lens), list(new), kind, dtype, page
        B = len(lens)
        need = [-(-n // page) for n in lens]
        self.pages = sum(need) + spare
        self.width = width or max(need + [1])
        pool = g.permutation(self.pages)
        self.table = np.full((B, self.width), -1, np.int64)
        at = 0
        shape = (self.pages, Hkv, page, K) if heads_first else (self.pages, page, Hkv, K)
        kc = torch.full(shape, float("nan"), dtype=t)
        vc = torch.full(shape[:3] + (V,), float("nan"), dtype=t)
        if heads_first:
            kc, vc = kc.permute(0, 2, 1, 3), vc.permute(0, 2, 1, 3)
        self.k, self.v = [], []
        for b in range(B):
            self.table[b, :need[b]] = pool[at:at + need[b]]
            at += need[b]
            k = torch.randn(lens[b], Hkv, K, generator=tg).to(t)
            v = torch.randn(lens[b], Hkv, V, generator=tg).to(t)
            for i in range(need[b]):
                n = min(page, lens[b] - i * page)
                kc[self.table[b, i], :n] = k[i * page:i * page + n]
                vc[self.table[b, i], :n] = v[i * page:i * page + n]
            self.k.append(k.double().numpy())
            self.v.append(v.double().numpy())
        self.rows = sum(new) + pad
        self.q = torch.randn(self.rows, H, K, generator=tg).to(t)
        self.starts = np.concatenate([[0], np.cumsum(new)])
        self.parents = None
        if kind is not None:
            self.parents = np.concatenate([tree(kind, n, g) for n in new] + [np.full(pad, -1)]).astype(np.int64)
        self.kc, self.vc, self.dev = kc.to(dev), vc.to(dev), dev

    def args(self):
        d = lambda x: None if x is None else torch.as_tensor(np.asarray(x, np.int64)).to(torch.int32).to(self.dev)
        return [self.q.to(self.dev), self.kc, self.vc, d(self.table), d(self.lens), d(self.starts)], d(self.parents)

    def run(self, **kw):
        a, p = self.args()
        o = htree_amd.draft_attention(*a, parents=p, **kw)
        torch.cuda.synchronize()
        return o

    def check(self, out, scale=None, holes=(), lens=None, odd=None):
        q = self.q.double().numpy()
        K = q.shape[2]
        scale = K ** -0.5 if scale is None else scale
        got = out.double().cpu().numpy()
        worst = 0.0
        for b, n in enumerate(self.new):
            s0 = self.starts[b]
            L = self.lens[b] if lens is None else lens[b]
            k, v = self.k[b][:L], self.v[b][:L]
            see = visible(self.kind, None if self.parents is None else self.parents[s0:s0 + n], n, L - n, L)
            for (bb, i) in holes:
                if bb == b:
                    see[:, i * self.page:(i + 1) * self.page] = False
            want, bar = reference(q[s0:s0 + n], k, v, see, scale, self.dtype)
            err = np.abs(got[s0:s0 + n] - want)
            bad = ~(err <= bar)
            assert not bad.any(), (
                f"request {b}: {int(bad.sum())} of {bad.size} outside, first {np.argwhere(bad)[0].tolist()}: "
                f"{got[s0:s0 + n][bad][0]} for {want[bad][0]} (bar {bar[bad][0]})")
            if err.size:
                worst = max(worst, float((err / bar).max()))
        return worst


HEADS = [(8, 1, 128, 128), (32, 2, 128, 128), (4, 4, 64, 64), (6, 2, 96, 80), (20, 1, 32, 64), (16, 2, 256, 256),
         (3, 1, 16, 8)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("H,Hkv,K,V", HEADS)
def test_single_tokens(dtype, H, Hkv, K, V):
    c = Case([1, 2, 15, 16, 17, 31, 33, 64, 65, 200, 0, 127, 128, 129], [1] * 10 + [0, 1, 1, 1], H, Hkv, K, V, dtype)
    c.check(c.run())


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("H,Hkv,K,V", HEADS)
@pytest.mark.parametrize("kind", ["tree", "star", None])
def test_drafted_tokens(dtype, H, Hkv, K, V, kind):
    """Trees, siblings and chains over contexts that end at and beside tile
    and page ends, none at all among them; requests without new tokens."""
    c = Case([5, 24, 40, 63, 64, 65, 96, 130, 16, 50], [5, 24, 8, 1, 16, 17, 3, 66, 0, 2], H, Hkv, K, V, dtype,
             kind=kind, seed=3)
    c.check(c.run())


@pytest.mark.parametrize("dtype,H,Hkv,K,V", [("bfloat16", 32, 2, 128, 128), ("bfloat16", 8, 1, 128, 128),
                                             ("float16", 8, 2, 64, 64), ("float32", 64, 4, 32, 32),
                                             ("bfloat16", 16, 2, 256, 256), ("float32", 4, 1, 128, 256),
                                             ("float32", 4, 2, 256, 32), ("float32", 40, 1, 64, 64)])
@pytest.mark.parametrize("kind,new", [(None, [1, 1, 1]), ("tree", [5, 24, 64]), (None, [300, 77, 1])])
def test_long_contexts_are_split(dtype, H, Hkv, K, V, kind, new):
    """Tables long enough that requests are split into chunks and joined: one
    long, one of a few tiles, one short."""
    c = Case([6001, 1500, 90], new, H, Hkv, K, V, dtype, kind=kind, page=32, seed=4)
    c.check(c.run())


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("heads_first", [False, True])
def test_pages_and_layouts(page, heads_first):
    c = Case([700, 1, 257, 256], [4, 1, 3, 40], 8, 2, 64, 64, "bfloat16", page=page, kind="tree",
             heads_first=heads_first, seed=5)
    c.check(c.run())


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("H,Hkv,K,V", HEADS + [(64, 1, 48, 128), (16, 1, 256, 200)])
@pytest.mark.parametrize("kind", ["tree", None])
def test_many_rows(dtype, H, Hkv, K, V, kind):
    """Requests of many rows (new tokens x heads of a group), ragged, without
    a cached token, split over their tokens; head dims that are not a
    kernel's among them."""
    c = Case([130, 300, 1400, 97], [130, 90, 200, 1], H, Hkv, K, V, dtype, kind=kind, seed=30)
    c.check(c.run())


def test_long_chunk_from_nothing():
    """A whole prompt: every row sees another number of tokens."""
    c = Case([1500], [1500], 4, 2, 32, 32, "bfloat16", seed=31)
    c.check(c.run())


def test_a_group_of_1024_heads():
    c = Case([70, 3], [2, 1], 1024, 1, 32, 32, "float16", kind="tree", seed=32)
    c.check(c.run())


def test_requests_that_share_pages():
    """A prefix in the same pages of two requests, and a table that names one
    page twice."""
    c = Case([96, 96, 40], [3, 5, 1], 8, 2, 64, 64, "bfloat16", kind="tree", seed=33)
    c.table[1, :3] = c.table[0, :3]
    c.table[2, 1] = c.table[2, 0]
    for x in (c.k, c.v):
        x[1][:48] = x[0][:48]
        x[2][16:32] = x[2][:16]
    c.check(c.run())


def test_rows_that_begin_later():
    """starts[0] > 0: the rows before it belong to no request."""
    c = Case([40, 70], [3, 2], 8, 2, 64, 64, "bfloat16", seed=34, pad=4)
    a, _ = c.args()
    out = torch.full((9, 8, 64), 9.0, dtype=torch.bfloat16, device=DEV)
    want = htree_amd.draft_attention(*a)
    a[0] = torch.cat([torch.zeros_like(a[0][:4]), a[0][:5]])
    a[5] = a[5] + 4
    htree_amd.draft_attention(*a, out=out)
    torch.cuda.synchronize()
    assert bool((out[:4] == 9.0).all()) and torch.equal(out[4:], want[:5])


@pytest.mark.parametrize("rows", [6, 400])
def test_damaged_lengths_stay_in_bounds(rows):
    """Starts and lengths that contradict each other (their indexes are
    replayed on the host too): rows outside what any request claims are left."""
    c = Case([200, 64, 90], [rows - 4, 2, 2], 8, 2, 64, 64, "bfloat16", seed=35, width=80)
    a, _ = c.args()
    for starts, lens in (([0, 3, 1, 5], [200, 64, 90]), ([2 ** 31 - 1, -2 ** 31, 3, 4], [200, 64, 90]),
                         ([1, 2, 3, 2 ** 31 - 1], [2 ** 31 - 1, -1, -2 ** 31]), ([0, 0, 0, 0], [5, 5, 5])):
        out = torch.full((rows, 8, 64), 9.0, dtype=torch.bfloat16, device=DEV)
        htree_amd.draft_attention(a[0], a[1], a[2], a[3], i32(lens), i32(starts), out=out)
        torch.cuda.synchronize()
        claimed = torch.zeros(rows, dtype=torch.bool)
        for s, e in zip(starts, starts[1:]):
            claimed[min(max(s, 0), rows):min(max(e, 0), rows)] = True
        assert bool((out[~claimed.to(DEV)] == 9.0).all())


def test_many_requests():
    g = np.random.default_rng(0)
    lens = g.integers(1, 300, 333)
    c = Case(lens, np.minimum(lens, g.integers(0, 4, 333)), 8, 2, 64, 64, "bfloat16", kind="tree", seed=6, width=70)
    c.check(c.run())


@pytest.mark.parametrize("scale", [0.0, -0.3, 5.0])
def test_scales(scale):
    c = Case([70, 130], [3, 40], 8, 2, 64, 64, "bfloat16", kind="tree", seed=7)
    c.check(c.run(scale=scale), scale=scale)


@pytest.mark.parametrize("width", [None, 200])
def test_holes_and_rows_that_see_nothing(width):
    """Table entries outside the cache hold no tokens; a request without any
    gives zeros."""
    c = Case([60, 40, 20, 2000], [2, 3, 4, 5], 8, 2, 64, 64, "bfloat16", kind="tree", seed=8, width=width)
    holes = [(0, 1), (1, 0), (1, 1), (1, 2), (2, 1), (3, 0), (3, 50), (3, 124)]
    for i, (b, p) in enumerate(holes):
        c.table[b, p] = (-1, c.pages, 2 ** 31 - 1, -2 ** 31)[i % 4]
    out = c.run()
    c.check(out, holes=holes)
    assert float(out[2:5].abs().max()) == 0.0


def test_lengths_past_the_table_and_below_the_new_tokens():
    """Tokens past the table's width are not there; with fewer tokens than
    new ones the first rows see nothing."""
    c = Case([64, 64, 64], [3, 5, 4], 8, 2, 64, 64, "bfloat16", seed=9, pad=0)
    a, p = c.args()
    a[4] = i32([70, 2, -5])
    o = htree_amd.draft_attention(*a)
    torch.cuda.synchronize()
    got = o.double().cpu().numpy()
    q = c.q.double().numpy()
    for b, (L, n) in enumerate(zip([70, 2, 0], c.new)):
        s0 = c.starts[b]
        see = np.arange(64)[None] <= (L - n + np.arange(n))[:, None]
        want, bar = reference(q[s0:s0 + n], c.k[b], c.v[b], see, 0.125, "bfloat16")
        assert np.all(np.abs(got[s0:s0 + n] - want) <= bar), b
    assert float(o[3:6].abs().max()) == 0.0 and float(o[8:].abs().max()) == 0.0


def test_parents_out_of_order_are_roots():
    c = Case([50, 50], [6, 6], 8, 2, 64, 64, "bfloat16", kind="tree", seed=10)
    c.parents = np.array([0, 5, 1, -9, 2 ** 31 - 1, 3, 7, 0, 2, 1, 3, 4])
    c.check(c.run())


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("K", [32, 64, 128, 256])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_branches_do_not_see_each_others_infinities(dtype, K, bad):
    """A drafted token with an infinite or NaN value or key reaches the rows
    that see it, and no others."""
    new = 20
    c = Case([70], [new], 4, 2, K, K, dtype, kind="tree", seed=11, spare=0)
    a, p = c.args()
    par = c.parents
    clean = htree_amd.draft_attention(*a, parents=p)
    tok, key = 7, 11
    for i, cache in ((tok, c.vc), (key, c.kc)):
        at = 70 - new + i
        cache[c.table[0, at // 16], at % 16, 1, K // 2] = bad
    out = htree_amd.draft_attention(*a, parents=p)
    torch.cuda.synchronize()
    see = visible("tree", par, new, 70 - new, 70)
    sv, sk = see[:, 50 + tok], see[:, 50 + key]
    assert 0 < sv.sum() < new and 0 < sk.sum() < new
    # A token with such a value joins the others' sum apart from the matrix
    # product, with P unrounded and in another order: rows that see it keep
    # their other dims to the bound of `reference` (each of the two results
    # is within it of the exact one), not to the bit.
    _, bar = reference(c.q.double().numpy(), c.k[0], c.v[0], see, K ** -0.5, dtype)
    bar = torch.as_tensor(bar, dtype=torch.float32, device=DEV)[:, 2:] * 1.0001
    for j in range(new):
        assert torch.equal(out[j, :2], clean[j, :2])          # the other KV head's
        x, y = out[j, 2:].float(), clean[j, 2:].float()
        if sk[j]:
            # an infinite score is NaN or a probability of 1; a NaN one NaN
            continue
        hit = torch.zeros(K, dtype=torch.bool, device=DEV)
        if sv[j]:
            hit[K // 2] = True
            assert not torch.isfinite(x[:, hit]).any()
            assert bool(((x - y).abs() <= 2 * bar[j])[:, ~hit].all())
        else:
            assert torch.equal(x, y)
        assert torch.isfinite(x[:, ~hit]).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("K,V", [(64, 64), (128, 96), (256, 256)])
def test_infinities_among_many_rows(dtype, K, V):
    """The same with many rows, several such tokens (one of them cached, in a
    tile with new ones) and pages missing."""
    new, L = 40, 110
    c = Case([L], [new], 16, 2, K, V, dtype, kind="tree", seed=36)
    c.table[0, 2] = -1
    a, p = c.args()
    clean = htree_amd.draft_attention(*a, parents=p)
    see = visible("tree", c.parents, new, L - new, L)
    see[:, 32:48] = False
    odd = [68, 75, 76, 90, 109]
    for i, at in enumerate(odd):
        c.vc[c.table[0, at // 16], at % 16, 1, i] = (float("inf"), float("nan"), -float("inf"))[i % 3]
    out = htree_amd.draft_attention(*a, parents=p)
    torch.cuda.synchronize()
    _, bar = reference(c.q.double().numpy(), c.k[0], c.v[0], see, K ** -0.5, dtype)
    bar = torch.as_tensor(bar, dtype=torch.float32, device=DEV)[:, 8:] * 1.0001
    assert torch.equal(out[:, :8], clean[:, :8])
    for j in range(new):
        x, y = out[j, 8:].float(), clean[j, 8:].float()
        hit = torch.zeros(V, dtype=torch.bool, device=DEV)
        for i, at in enumerate(odd):
            hit[i] = bool(see[j, at])
        assert not torch.isfinite(x[:, hit]).any()
        assert bool(((x - y).abs() <= 2 * bar[j])[:, ~hit].all())
        if not hit.any():
            assert torch.equal(x, y)


def test_rows_behind_the_last_are_left():
    c = Case([40, 1500], [3, 2], 8, 2, 64, 64, "bfloat16", seed=12, pad=7)
    out = torch.full((12, 8, 64), 9.0, dtype=torch.bfloat16, device=DEV)
    assert c.run(out=out) is out
    c.check(out)
    assert bool((out[5:] == 9.0).all())


def test_strided_queries_and_tables():
    c = Case([40, 1500], [3, 2], 8, 2, 64, 64, "bfloat16", kind="tree", seed=13)
    a, p = c.args()
    want = htree_amd.draft_attention(*a, parents=p)
    fused = torch.zeros(5, 12, 64, dtype=torch.bfloat16, device=DEV)
    fused[:, :8] = a[0]
    wide = torch.full((2, 200), -5, dtype=torch.int32, device=DEV)
    wide[:, :a[3].shape[1]] = a[3]
    shifted = torch.empty(5 * 8 * 64 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(5, 8, 64)
    shifted.copy_(a[0])
    for q in (fused[:, :8], shifted, a[0].transpose(0, 2).contiguous().transpose(0, 2)):
        got = htree_amd.draft_attention(q, a[1], a[2], wide[:, :a[3].shape[1]], a[4], a[5], parents=p)
        assert torch.equal(got, want)


def test_cache_past_32_bits():
    """Keys and values beyond 2^32 bytes into the cache."""
    c = Case([50, 1200], [2, 3], 32, 16, 128, 128, "bfloat16", kind="tree", seed=14, spare=0)
    pages = 70000
    big = [torch.empty(pages, 16, 16, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    far = np.arange(pages - c.pages, pages)
    for x, y in zip(big, (c.kc, c.vc)):
        assert x.numel() * 2 > 2 ** 32
        x[pages - c.pages:] = y
    c.table = np.where(c.table >= 0, far[np.maximum(c.table, 0)], -1)
    c.kc, c.vc = big
    c.check(c.run())


def test_same_results_twice_and_alone():
    """Bit for bit, and a call's results do not depend on what ran before."""
    c = Case([3000, 200, 17], [8, 1, 4], 32, 2, 128, 128, "bfloat16", kind="tree", seed=15)
    a = c.run()
    Case([900], [5], 32, 2, 128, 128, "bfloat16", seed=16).run()
    assert torch.equal(a, c.run())


def test_streams_and_graphs():
    """On another stream, and captured: two graphs and eager calls in turn,
    replayed over lengths that change between the replays."""
    cs = [Case([3000, 200, 64], [8, 1, 4], 32, 2, 128, 128, "bfloat16", kind="tree", seed=s) for s in (17, 18)]
    want = [c.run() for c in cs]
    side = torch.cuda.Stream()
    held = [c.args() for c in cs]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = [htree_amd.draft_attention(*a, parents=p) for a, p in held]
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    graphs, outs = [], []
    for a, p in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(htree_amd.draft_attention(*a, parents=p))
        graphs.append(g)
    shorter = [2000, 100, 33]
    for rep in range(4):
        for i in (0, 1):
            c, (a, p) = cs[i], held[i]
            lens = c.lens if rep % 2 == 0 else shorter
            a[4].copy_(i32(lens))
            outs[i].fill_(5.0)
            graphs[i].replay()
            eager = htree_amd.draft_attention(*a, parents=p)
            torch.cuda.synchronize()
            assert torch.equal(outs[i], eager)
            c.check(outs[i], lens=lens)


def test_two_calls_at_once():
    """Two streams at the same time, each with a workspace of its own."""
    cs = [Case([5000, 200], [8, 1], 32, 2, 128, 128, "bfloat16", kind="tree", seed=s) for s in (19, 20)]
    want = [c.run() for c in cs]
    held = [c.args() for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(htree_amd.draft_attention(*held[i][0], parents=held[i][1]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in (0, 1) for x in got[i])


def test_empty_calls():
    c = Case([40], [0], 8, 2, 64, 64, "bfloat16", seed=21)
    assert c.run().shape == (0, 8, 64)
    e = Case([40], [2], 8, 2, 64, 64, "bfloat16", seed=21)
    a, _ = e.args()
    out = torch.full((2, 8, 64), 3.0, dtype=torch.bfloat16, device=DEV)
    htree_amd.draft_attention(a[0], a[1], a[2], a[3][:0], a[4][:0], a[5][:1], out=out)
    assert bool((out == 3.0).all())
    got = htree_amd.draft_attention(a[0], a[1], a[2], a[3][:, :0], a[4], a[5])  # a table of no pages
    assert float(got.abs().max()) == 0.0


def test_refusals():
    c = Case([40], [2], 8, 2, 64, 64, "bfloat16", seed=22)
    a, _ = c.args()
    da = htree_amd.draft_attention
    q, kc, vc, tab, lens, starts = a
    bad = [
        lambda: da(q[:, :7], kc, vc, tab, lens, starts), lambda: da(q[..., :32], kc, vc, tab, lens, starts),
        lambda: da(q.float(), kc, vc, tab, lens, starts), lambda: da(q, kc, vc, tab.long(), lens, starts),
        lambda: da(q, kc, vc, tab, lens.long(), starts), lambda: da(q, kc, vc, tab, lens, starts[:1]),
        lambda: da(q, kc, vc[:1], tab, lens, starts), lambda: da(q, kc, vc, tab, lens, starts, parents=lens),
        lambda: da(q.cpu(), kc, vc, tab, lens, starts), lambda: da(q, kc, vc, tab.cpu(), lens, starts),
        lambda: da(q, kc[:, :8], vc[:, :8], tab, lens, starts),
        lambda: da(q, kc, vc, tab, lens, starts, out=torch.empty(2, 8, 32, device=DEV)),
        lambda: da(q.clone().requires_grad_(), kc, vc, tab, lens, starts),
        lambda: da(q[0], kc, vc, tab, lens, starts), lambda: da(q, kc, vc, tab, lens, starts, out=q),
        lambda: da(q, kc, vc, tab, lens, starts, scale=float("nan")),
        lambda: da(q, kc, vc, tab, lens, starts, scale=float("inf")),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(AssertionError):
            call()
            print("not refused:", i)


# ------------------------------------------------------------ run together
def test_continues_htree_forward():
    """Up to max_top_nodes tokens the tree has one level, and the rows of
    htree_forward are those of the cache: a prompt written into pages, then
    its last tokens as a chain, a chunk and one by one.  Both round the same
    inputs (bf16) but the cache rounds rotated keys and queries once more:
    half a step each of |q||k| scale in a score, and P's and the output's
    half steps on either side."""
    B, T, H, Hkv, D, page = 2, 500, 8, 2, 128, 16
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(B, T, h, D, generator=g).bfloat16().to(DEV) for h in (H, Hkv, Hkv))
    want = htree_amd.htree_forward(q, k, v, 16, 1024, 64).double()
    cos, sin = htree_amd.rope_cache(D, T, 10000.0, DEV)
    pages = 80
    kc, vc = (torch.full((pages, page, Hkv, D), float("nan"), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    table = torch.full((B, 40), -1, dtype=torch.int32, device=DEV)
    free = torch.randperm(pages, generator=g).to(torch.int32).to(DEV)
    ctx = i32([0] * B)
    half = 2.0 ** -8
    score = 2 * half * (q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max()) * D ** -0.5
    done = 0
    for n, chain in ((401, False), (1, False), (40, True), (1, True), (57, False)):
        new = i32([n] * B)
        rows = n * B + 3
        par = torch.cat([torch.arange(n) - 1] * B + [torch.full((3,), -1)]).to(torch.int32).to(DEV)
        t = htree_amd.page_tables(ctx, new, table, free, page, pages, rows, parents=par if chain else None)
        free = free[int(t.pages_used):].contiguous()
        pick = lambda x: torch.cat([x[:, done:done + n].reshape(B * n, -1, D), x[0, :3]])
        qr = htree_amd.cache_append(pick(k), pick(v), kc, vc, t.slots, q=pick(q), positions=t.positions, cos=cos, sin=sin)
        out = htree_amd.draft_attention(qr, kc, vc, table, t.lens, t.starts, parents=par if chain else None)
        got = out[:B * n].view(B, n, H, D).double()
        w = want[:, done:done + n]
        vmax = v.double().abs().max()
        # |A| <= max |v|; the average of iid values is far below it
        bar = vmax * (torch.expm1(2 * score) + 2 * half) + 2 * half * w.abs()
        assert bool(((got - w).abs() <= bar).all())
        # and in the mean as close as two roundings of each side allow
        rel = float((got - w).norm() / w.norm())
        assert rel < 4 * half, rel
        ctx, done = t.lens.clone(), done + n
    assert done == T


def test_a_captured_step_of_serving():
    """Tables, append and attention of drafted trees in one graph, replayed
    step after step; between the replays a branch is accepted, written to
    where it stays, and the pages it took leave the pool."""
    B, H, Hkv, D, page, n, pages = 3, 8, 2, 64, 16, 9, 64
    dt = torch.bfloat16
    g = torch.Generator().manual_seed(1)
    rng = np.random.default_rng(1)
    cos, sin = htree_amd.rope_cache(D, 300, 10000.0, DEV)
    kc, vc = (torch.full((pages, page, Hkv, D), float("nan"), dtype=dt, device=DEV) for _ in range(2))
    table = torch.full((B, 20), -1, dtype=torch.int32, device=DEV)
    pool = torch.randperm(pages, generator=g).to(torch.int32).to(DEV)
    free = pool.clone()
    ctx, new = i32([0] * B), i32([n] * B)
    rows = B * n
    par = i32(np.concatenate([tree("tree", n, rng) for _ in range(B)]))
    qkv = torch.zeros(rows, H + 2 * Hkv, D, dtype=dt, device=DEV)

    def step():
        t = htree_amd.page_tables(ctx, new, table, free, page, pages, rows, parents=par)
        qr = htree_amd.cache_append(qkv[:, H:H + Hkv], qkv[:, H + Hkv:], kc, vc, t.slots, q=qkv[:, :H],
                                    positions=t.positions, cos=cos, sin=sin)
        return t, qr, htree_amd.draft_attention(qr, kc, vc, table, t.lens, t.starts, parents=par)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t, qr, out = step()
    hist = [(np.zeros((0, Hkv, D)), np.zeros((0, Hkv, D))) for _ in range(B)]
    for rep in range(6):
        qkv.copy_(torch.randn(rows, H + 2 * Hkv, D, generator=g).to(dt))
        parents = np.concatenate([tree("tree", n, rng) for _ in range(B)])
        par.copy_(i32(parents))
        graph.replay()
        eager = htree_amd.draft_attention(qr, kc, vc, table, t.lens, t.starts, parents=par)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        slots = t.slots.cpu().numpy()
        got = out.double().cpu().numpy()
        kn = kc.double().cpu().numpy().reshape(-1, Hkv, D)[slots]
        vn = vc.double().cpu().numpy().reshape(-1, Hkv, D)[slots]
        keep, kept_new = [], []
        for b in range(B):
            k = np.concatenate([hist[b][0], kn[b * n:(b + 1) * n]])
            v = np.concatenate([hist[b][1], vn[b * n:(b + 1) * n]])
            L = len(k)
            p = parents[b * n:(b + 1) * n]
            see = visible("tree", p, n, L - n, L)
            qb = qr.double().cpu().numpy()[b * n:(b + 1) * n]
            want, bar = reference(qb, k, v, see, D ** -0.5, "bfloat16")
            assert np.all(np.abs(got[b * n:(b + 1) * n] - want) <= bar), (rep, b)
            path, a = [], int(rng.integers(0, n))
            while a >= 0:
                path.append(b * n + a)
                a = int(p[a])
            path.reverse()
            keep += path
            kept_new.append(len(path))
            hist[b] = (np.concatenate([hist[b][0], kn[path]]), np.concatenate([hist[b][1], vn[path]]))
        # the accepted branches, rotated already, to the slots where they stay
        x, y = kc.view(-1, Hkv, D)[t.slots[keep]], vc.view(-1, Hkv, D)[t.slots[keep]]
        first = np.concatenate([np.arange(m) for m in kept_new]) + np.repeat(np.arange(B) * n, kept_new)
        htree_amd.cache_append(x, y, kc, vc, t.slots[torch.as_tensor(first).to(DEV)].contiguous())
        ctx.add_(i32(kept_new))
        # pages that hold tokens now leave the pool; the others are free again
        used = table[torch.arange(20, device=DEV) < ((ctx + page - 1) // page)[:, None]]
        left = pool[~torch.isin(pool, used)]
        free.fill_(-1)
        free[:left.numel()] = left
        assert [len(h[0]) for h in hist] == ctx.tolist()

"""GPU tests of keep_drafts, copy_pages, fork_requests and unused_pages
against their definitions, token by token.  What they move keeps its bits;
everything is compared whole, so that nothing else may change."""
import numpy as np
import pytest
import torch

import htree_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def i32(x):
    return torch.as_tensor(np.asarray(x, np.int64)).to(torch.int32).to(DEV)


def caches(layout, layers, pages, page, H, K, V, dtype, seed):
    """Key and value caches of a layout, and each layer's as [pages, page, H, D]."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *n: torch.randn(*n, generator=g, device=DEV).to(DT[dtype])
    if layout == "one":
        k, v = rand(pages, page, H, K), rand(pages, page, H, V)
        return k, v, [k], [v]
    if layout == "stacked":
        k, v = rand(layers, pages, page, H, K), rand(layers, pages, page, H, V)
        return k, v, list(k), list(v)
    if layout == "list":
        k, v = [rand(pages, page, H, K) for _ in range(layers)], [rand(pages, page, H, V) for _ in range(layers)]
        return k, v, k, v
    if layout == "heads first":  # a permuted cache, layers inside pages
        k, v = (rand(pages, layers, H, page, D).permute(1, 0, 3, 2, 4) for D in (K, V))
        return k, v, list(k), list(v)
    assert layout == "beside"  # keys beside values in one buffer, gaps between heads
    both = rand(pages, page, layers, H, K + V + 16).permute(2, 0, 1, 3, 4)
    k, v = both[..., :K], both[..., K:K + V]
    return k, v, list(k), list(v)


LAYOUTS = [("one", 1, 16, 2, 128, 128, "bfloat16"), ("stacked", 5, 16, 3, 64, 32, "float16"),
           ("list", 3, 64, 4, 32, 32, "float32"), ("heads first", 4, 32, 2, 96, 96, "bfloat16"),
           ("beside", 2, 16, 5, 8, 16, "bfloat16"), ("stacked", 70, 16, 1, 8, 8, "float16"),
           ("list", 129, 16, 1, 4, 8, "float32"), ("one", 1, 16, 40, 256, 256, "float32")]


def steps(B, most, page, g):
    """New tokens' slots over a shuffled pool, and which of them are kept."""
    new = g.integers(0, most + 1, B)
    new[0] = most
    ctx = g.integers(0, 2 * page, B)
    had = [-(-(c + n) // page) for c, n in zip(ctx, new)]
    pool = g.permutation(sum(had) + 3)
    starts = np.concatenate([[0], np.cumsum(new)])
    rows = int(starts[-1]) + 2
    slots, path, kept = np.full(rows, -1, np.int64), np.full(rows, -1), np.zeros(B, int)
    at = 0
    for b in range(B):
        for j in range(new[b]):
            p = ctx[b] + j
            slots[starts[b] + j] = pool[at + p // page] * page + p % page
        at += had[b]
        kept[b] = g.integers(0, new[b] + 1)
        path[starts[b]:starts[b] + kept[b]] = np.sort(g.choice(new[b], kept[b], replace=False)) if new[b] else []
    return slots, starts, path, kept, len(pool)


def moved(x, pairs, page):
    """x [pages, page, H, D] with the rows of (from, to) moved, each read first."""
    y = x.clone()
    for a, b in pairs:
        y[b // page, b % page] = x[a // page, a % page]
    return y


@pytest.mark.parametrize("layout,layers,page,H,K,V,dtype", LAYOUTS)
@pytest.mark.parametrize("B,most", [(1, 1), (3, 24), (7, 70)])
def test_keep_drafts(layout, layers, page, H, K, V, dtype, B, most):
    g = np.random.default_rng(B + layers)
    slots, starts, path, kept, pages = steps(B, most, page, g)
    k, v, ks, vs = caches(layout, layers, pages, page, H, K, V, dtype, 1)
    pairs = [(slots[starts[b] + path[starts[b] + j]], slots[starts[b] + j]) for b in range(B) for j in range(kept[b])]
    want = [moved(x, pairs, page) for x in ks + vs]
    htree_amd.keep_drafts(k, v, torch.as_tensor(slots).to(DEV), i32(starts), i32(path), i32(kept))
    for x, y in zip(ks + vs, want):
        assert torch.equal(x, y)


def test_keep_drafts_of_damaged_lists_stays_inside():
    """Slots, paths, starts and counts of any values: rows outside the cache's
    view stay as they were, and a list that does not ascend moves nothing to
    where it should not go."""
    g = np.random.default_rng(4)
    page, pages, B, rows = 16, 6, 4, 40
    big_k, big_v = (torch.randn(pages + 4, page, 2, 64, device=DEV).bfloat16() for _ in range(2))
    before = big_k.clone(), big_v.clone()
    k, v = big_k[2:-2], big_v[2:-2]
    for seed in range(20):
        g = np.random.default_rng(seed)
        wild = lambda n, lo, hi: np.where(g.random(n) < 0.3, g.integers(-2 ** 31, 2 ** 31, n), g.integers(lo, hi, n))
        slots = torch.as_tensor(np.where(g.random(rows) < 0.3, g.integers(-2 ** 62, 2 ** 62, rows),
                                         g.integers(0, pages * page, rows))).to(DEV)
        htree_amd.keep_drafts(k, v, slots, i32(wild(B + 1, 0, rows)), i32(wild(rows, 0, 12)), i32(wild(B, 0, 12)))
    for x, y in ((big_k, before[0]), (big_v, before[1])):
        assert torch.equal(x[:2], y[:2]) and torch.equal(x[-2:], y[-2:])
    # not ascending: only what comes from behind its place moves
    x = k.clone()
    htree_amd.keep_drafts(k, v, torch.arange(8, device=DEV), i32([0, 8]), i32([3, 0, 1, 2, 4, 9, -1, 7]), i32([8]))
    assert torch.equal(k, moved(x, [(3, 0)], page))


@pytest.mark.parametrize("layout,layers,page,H,K,V,dtype", LAYOUTS)
@pytest.mark.parametrize("whole", [False, True])
def test_copy_pages(layout, layers, page, H, K, V, dtype, whole):
    g = np.random.default_rng(layers)
    pages, n = 23, 9
    perm = g.permutation(pages)
    frm, to, count = perm[:n].copy(), perm[n:2 * n].copy(), g.integers(0, page + 1, n)
    count[0], count[1] = page, 0
    frm[2], to[3], frm[4], to[5], frm[6], count[7] = -1, -1, pages, 2 ** 31 - 1, -2 ** 31, -5
    frm[8] = frm[0]  # one page to several
    k, v, ks, vs = caches(layout, layers, pages, page, H, K, V, dtype, 2)
    pairs = [(a * page + t, b * page + t) for a, b, c in zip(frm, to, count) if 0 <= a < pages and 0 <= b < pages
             for t in range(page if whole else max(c, 0))]
    want = [moved(x, pairs, page) for x in ks + vs]
    htree_amd.copy_pages(k, v, i32(frm), i32(to), None if whole else i32(count))
    for x, y in zip(ks + vs, want):
        assert torch.equal(x, y)


def plain_fork(table, lens, source, free, page, pages):
    width, used, had = table.shape[1], 0, set()
    out, o_lens, frm, to, count = [], [], [], [], []
    for s in source:
        row, L, a, b, c = np.full(width, -1), 0, -1, -1, 0
        if 0 <= s < len(lens):
            L = max(int(lens[s]), 0)
            live = min(-(-L // page), width)
            row[:live] = table[s, :live]
            if L % page and L // page < width and s in had:
                pg = free[used] if used < len(free) and 0 <= free[used] < pages else -1
                used += 1
                old = row[L // page]
                row[L // page] = pg
                if pg >= 0 and 0 <= old < pages:
                    a, b, c = old, pg, L % page
            had.add(s)
        out.append(row), o_lens.append(L), frm.append(a), to.append(b), count.append(c)
    return np.array(out).reshape(-1, width), o_lens, frm, to, count, [used]


@pytest.mark.parametrize("B,n,width,page", [(1, 8, 5, 16), (5, 5, 9, 16), (4, 1, 1, 32), (64, 256, 30, 16), (300, 700, 3, 64),
                                            (4096, 4096, 2, 16), (2, 3, 3000, 16), (3, 4, 6, 1), (3, 0, 4, 16), (0, 3, 4, 16)])
def test_fork_requests(B, n, width, page):
    for seed in range(3):
        g = np.random.default_rng(seed + B)
        pages = max(B * width + n, 1)
        lens = g.integers(0, width * page + 1, B)
        table = g.permutation(pages)[:B * width].reshape(B, width)
        source = g.integers(0, max(B, 1), n) if seed else np.arange(n) % max(B, 1)
        if seed == 2:  # holes, requests of none, lengths past the table and below zero
            source[g.random(n) < 0.3] = g.choice([-1, B, 2 ** 31 - 1])
            table[g.random((B, width)) < 0.2] = g.choice([-1, pages, -2 ** 31])
            lens[g.random(B) < 0.2] = g.choice([-7, 2 ** 31 - 1, width * page + 1])
        free = g.permutation(pages)[:max(n // 2, 1) if seed == 2 else n]
        want = plain_fork(table, lens, source, free, page, pages)
        wide = torch.full((B, width + 3), 5, dtype=torch.int32, device=DEV)
        wide[:, :width] = i32(table).view(B, width)
        f = htree_amd.fork_requests(wide[:, :width], i32(lens), i32(source), i32(free), page, pages)
        for name, a, b in zip(f._fields, f, want):
            assert np.array_equal(a.cpu().numpy().reshape(-1), np.asarray(b).reshape(-1)), (name, seed)
        assert f.block_table.shape == (n, width)


def test_fork_writes_where_it_is_told():
    o = htree_amd.Forked(torch.full((3, 10), -9, dtype=torch.int32, device=DEV)[:, :4],
                         *(torch.full((m,), -9, dtype=torch.int32, device=DEV) for m in (3, 3, 3, 3, 1)))
    table, lens = i32([[4, 5, 6, -1], [7, -1, -1, -1]]), i32([40, 16])
    f = htree_amd.fork_requests(table, lens, i32([0, 1, 0]), i32([9]), 16, 12, out=o)
    assert f is o and o.block_table.tolist() == [[4, 5, 6, -1], [7, -1, -1, -1], [4, 5, 9, -1]]
    assert o.lens.tolist() == [40, 16, 40] and o.copy_from.tolist() == [-1, -1, 6] and o.copy_to.tolist() == [-1, -1, 9]
    assert o.copy_tokens.tolist() == [0, 0, 8] and o.pages_used.tolist() == [1]


def check_unused(table, lens, page, pages, held=None):
    used = {int(x) for row, L in zip(table, lens) for x in row[:max(0, -(-int(L) // page))]}  # (others than pages: no matter)
    used |= set() if held is None else {int(x) for x in held}
    want = np.array([p for p in range(pages) if p not in used], int)
    u = htree_amd.unused_pages(i32(table), i32(lens), page, pages,
                               held=None if held is None else i32(held))
    got = u.pages.cpu().numpy()
    assert int(u.count) == len(want) and np.array_equal(got[:len(want)], want) and (got[len(want):] == -1).all()


@pytest.mark.parametrize("B,width,page,pages", [(1, 1, 16, 1), (3, 20, 16, 100), (7, 300, 64, 4096), (7, 300, 64, 4097),
                                                (64, 1100, 16, 100000), (4096, 3, 16, 20000), (2, 40000, 16, 70001),
                                                (300, 3000, 16, 9000), (20, 1000, 16, 262144), (3, 2000, 64, 250001), (256, 200, 16, 131073),
                                                (0, 5, 16, 33), (4, 5, 1, 16), (5, 0, 16, 50), (300, 40, 16, 1 << 21)])
def test_unused_pages(B, width, page, pages):
    for seed in range(2):
        g = np.random.default_rng(seed + width)
        table, lens = g.integers(0, pages, (B, width)), g.integers(0, width * page + 1, B)
        held = g.integers(0, pages, 37) if seed else None
        if seed:  # entries and lengths of any values
            table[g.random((B, width)) < 0.2] = g.choice([-1, pages, 2 ** 31 - 1, -2 ** 31])
            lens[g.random(B) < 0.2] = g.choice([-1, 2 ** 31 - 1, 0])
            held[:4] = [-1, pages, 2 ** 31 - 1, -2 ** 31]
        check_unused(table, lens, page, pages, held)


def test_all_or_no_pages_unused():
    check_unused(np.arange(8192).reshape(2, 4096), [65536, 65536], 16, 8192)
    check_unused(np.arange(8192).reshape(2, 4096), [0, 0], 16, 8192)
    check_unused(np.arange(8192).reshape(2, 4096), [0, 0], 16, 8192, held=np.arange(8191, -1, -1))
    u = htree_amd.unused_pages(i32(np.zeros((1, 3))), i32([5]), 16, 0)
    assert int(u.count) == 0 and u.pages.numel() == 0


def test_past_32_bits():
    """Moves and copies between both ends of a cache of more than 2^32 bytes."""
    pages = 70000
    k = torch.empty(pages, 16, 16, 128, dtype=torch.bfloat16, device=DEV)
    v = torch.empty(pages, 16, 16, 128, dtype=torch.bfloat16, device=DEV)
    assert k.numel() * 2 > 2 ** 32
    ends = torch.randn(2, 2, 16, 16, 128, device=DEV).bfloat16()
    k[0], k[-1], v[0], v[-1] = ends[0, 0], ends[0, 1], ends[1, 0], ends[1, 1]
    htree_amd.copy_pages(k, v, i32([pages - 1, 0]), i32([1, pages - 2]), i32([16, 7]))
    assert torch.equal(k[1], ends[0, 1]) and torch.equal(v[1], ends[1, 1])
    assert torch.equal(k[-2, :7], ends[0, 0, :7]) and torch.equal(v[-2, :7], ends[1, 0, :7])
    slots = torch.tensor([5, pages * 16 - 3, pages * 8], device=DEV)
    htree_amd.keep_drafts(k, v, slots, i32([0, 3]), i32([1, -1, -1]), i32([1]))
    assert torch.equal(k[0, 5], ends[0, 1, 13]) and torch.equal(v[0, 5], ends[1, 1, 13])


def test_refusals():
    f = lambda *n, t=torch.bfloat16: torch.zeros(n, dtype=t, device=DEV)
    I, L = torch.int32, torch.int64
    k, v = f(4, 16, 2, 64), f(4, 16, 2, 64)
    lists = (f(3, t=L), f(2, t=I), f(3, t=I), f(1, t=I))
    keep = lambda a=k, b=v, s=lists: htree_amd.keep_drafts(a, b, *s)
    copy = lambda a=k, b=v, x=f(2, t=I), y=f(2, t=I), z=None: htree_amd.copy_pages(a, b, x, y, z)
    fork = lambda t=f(2, 3, t=I), n=f(2, t=I), s=f(4, t=I), r=f(5, t=I), p=16, m=9, **kw: \
        htree_amd.fork_requests(t, n, s, r, p, m, **kw)
    unused = lambda t=f(2, 3, t=I), n=f(2, t=I), p=16, m=9, **kw: htree_amd.unused_pages(t, n, p, m, **kw)
    keep(), copy(), fork(), unused()
    swap = lambda i, x: tuple(x if j == i else y for j, y in enumerate(lists))
    out, uout = fork(), unused()
    bad = [lambda: keep(k, k), lambda: keep([k, k], [v, f(4, 16, 2, 64)]), lambda: keep([k], [v, v]),
           lambda: keep([], []), lambda: keep([k, f(5, 16, 2, 64)], [v, v]), lambda: keep(k.float(), v),
           lambda: keep(k[:1].expand(4, 16, 2, 64), v), lambda: keep(f(1, 4, 16, 2, 64).expand(3, 4, 16, 2, 64), f(3, 4, 16, 2, 64)),
           lambda: keep(f(4, 16, 2, 60), f(4, 16, 2, 60)), lambda: keep(f(4, 8, 2, 64), f(4, 8, 2, 64)),
           lambda: keep(k.cpu(), v.cpu()), lambda: keep(k.clone().requires_grad_(), v), lambda: keep(f(16, 2, 64), f(16, 2, 64)),
           lambda: keep(f(4 * 16 * 2 * 64 + 8)[4:-4].view(4, 16, 2, 64), v),
           lambda: keep(k, v.double()), lambda: keep(s=swap(0, f(3, t=I))), lambda: keep(s=swap(1, f(3, t=I))),
           lambda: keep(s=swap(2, f(2, t=I))), lambda: keep(s=swap(3, f(1, t=L))), lambda: keep(s=swap(3, f(4097, t=I))),
           lambda: copy(x=f(2, t=L)), lambda: copy(y=f(3, t=I)), lambda: copy(z=f(3, t=I)), lambda: copy(x=f(2, 1, t=I)),
           lambda: copy(k, v.cpu()), lambda: copy([k, v], [v, k]),
           lambda: fork(p=12), lambda: fork(m=-1), lambda: fork(n=f(3, t=I)), lambda: fork(s=f(4, t=L)),
           lambda: fork(s=f(4097, t=I)), lambda: fork(r=f(5, 1, t=I)), lambda: fork(t=f(3, 2, t=I).t()),
           lambda: fork(out=out._replace(lens=f(3, t=I))), lambda: fork(n=out.lens[:2], out=out),
           lambda: fork(out=out._replace(block_table=f(4, 2, t=I))), lambda: fork(t=out.block_table[:2], out=out),
           lambda: fork(out=out._replace(copy_to=out.copy_from)), lambda: unused(p=0), lambda: unused(p=48), lambda: unused(m=2 ** 31),
           lambda: unused(held=f(3, t=L)), lambda: unused(held=f(3, 1, t=I)), lambda: unused(n=f(1, t=I)),
           lambda: unused(out=uout._replace(pages=f(8, t=I))), lambda: unused(held=uout.pages, out=uout),
           lambda: unused(out=uout._replace(count=uout.pages[:1])), lambda: unused(t=f(2, 3, t=I).cpu())]
    for i, call in enumerate(bad):
        with pytest.raises(AssertionError):
            call()
            print("not refused:", i)

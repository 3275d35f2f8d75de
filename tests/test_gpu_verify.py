"""GPU tests of verify_drafts against the walk written out in 64 bits.  Its
answers are whole numbers and have to be equal: sums of the two differ by
about 1e-15 of the mass, so a draw or a test falls between them with a chance
of 1e-11 a token.  Probabilities that are multiples of 2^-10, whose sums are
exact in any order, meet the borders themselves."""
import numpy as np
import pytest
import torch

import htree_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def mass(x):
    return np.where(np.isfinite(x) & (x > 0), x, 0.0)


def positive(u):
    return u if u > 0 else 0.0


def walk(p, q, tokens, starts, parents, uniforms, draws):
    """The definition, request by request."""
    p = mass(np.asarray(p, np.float64))
    q = None if q is None else mass(np.asarray(q, np.float64))
    rows, V = p.shape
    B = len(starts) - 1
    kept, path, nxt = np.zeros(B, int), np.full(rows, -1), np.full(B, -1)
    for b in range(B):
        s0, n = starts[b], min(starts[b + 1] - starts[b], 1024)
        if n <= 0:
            continue
        up = [-1] * n
        for j in range(n):
            a = j - 1 if parents is None else parents[s0 + j]
            if 0 <= a < j and 0 <= tokens[s0 + j] < V:
                up[j] = a
        node, keep = 0, [0]
        while True:
            r, T, S, a, hit = s0 + node, p[s0 + node].copy(), 1.0, 0.0, -1
            for c in range(node + 1, n):
                if up[c] != node:
                    continue
                x, u = tokens[s0 + c], positive(float(uniforms[s0 + c]))
                if u * S * (1.0 if q is None else q[r, x]) < T[x]:
                    hit = c
                    break
                if q is None:
                    S, T[x] = S - T[x], 0.0
                else:
                    a += S
                    T = np.maximum(p[r] - a * q[r], 0)
                    S = T.sum()
            if hit < 0:
                break
            node = hit
            keep.append(node)
        kept[b], path[s0:s0 + len(keep)] = len(keep), keep
        if not T.sum() > 0:
            T = p[r]
        if T.sum() > 0:
            C = T.cumsum()
            nxt[b] = min(np.searchsorted(C, positive(float(draws[b])) * C[-1], side="right"), np.nonzero(T)[0].max())
    return kept, path, nxt


def check(p, q, tokens, starts, parents, uniforms, draws, **kw):
    i32 = lambda x: None if x is None else torch.as_tensor(np.asarray(x, np.int32)).to(DEV)
    f32 = lambda x: torch.as_tensor(np.asarray(x, np.float32)).to(DEV)
    p, q = p.to(DEV), None if q is None else q.to(DEV)
    want = walk(p.double().cpu().numpy(), None if q is None else q.double().cpu().numpy(), tokens, starts, parents,
                np.asarray(uniforms, np.float32), np.asarray(draws, np.float32))
    got = htree_amd.verify_drafts(p, torch.as_tensor(np.asarray(tokens, np.int64)).to(DEV), i32(starts), f32(uniforms),
                                  f32(draws), draft_probs=q, parents=i32(parents), **kw)
    for name, a, b in zip(got._fields, got, want):
        assert np.array_equal(a.cpu().numpy(), b), (name, a.cpu().numpy()[:20], b[:20])
    return want


def random_tree(n, g):
    return np.array([-1] + [max(0, j - 1 - int(g.integers(0, 5))) for j in range(1, n)])[:n]


def case(new, V, dtype, tree, drawn, seed, sharp=4.0, grid=None):
    """grid: probabilities in whole multiples of 1 / grid, numbers of draws too."""
    g = np.random.default_rng(seed)
    t = torch.Generator().manual_seed(seed)
    starts = np.concatenate([[0], np.cumsum(new)])
    rows = int(starts[-1])
    parents = np.concatenate([random_tree(n, g) for n in new] + [[]]).astype(int) if tree else None
    logits = torch.randn(rows, V, generator=t) * sharp
    p, q = torch.softmax(logits, -1), torch.softmax(logits + 0.7 * torch.randn(rows, V, generator=t), -1)
    u, d = g.random(rows, dtype=np.float32), g.random(len(new), dtype=np.float32)
    if grid:
        p, q = (p * grid).round() / grid, (q * grid).round() / grid
        u, d = np.floor(u * 8) / 8, np.floor(d * 8) / 8
    p, q = p.to(DT[dtype]), q.to(DT[dtype])
    tokens = np.zeros(rows, int)
    qn = q.double().numpy()
    for b in range(len(new)):
        for j in range(1, new[b]):
            up = starts[b] + (j - 1 if parents is None else parents[starts[b] + j])
            if drawn and qn[up].sum() > 0:
                tokens[starts[b] + j] = g.choice(V, p=qn[up] / qn[up].sum())
            else:
                tokens[starts[b] + j] = np.argsort(-qn[up])[g.integers(0, min(4, V))]
    return p, q if drawn else None, tokens, starts, parents, u, d


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("new,V,dtype", [
    ([6], 32000, "float32"), ([1, 2, 3], 1, "float32"), ([24] * 5, 7, "bfloat16"), ([2, 9, 1, 30], 8192, "float16"),
    ([5, 5], 8193, "float32"), ([64], 16385, "bfloat16"), ([65, 3], 777, "float32"), ([3] * 70, 301, "bfloat16"),
    ([0, 4, 0, 5, 0], 1001, "float32"), ([200, 1], 50, "float16"), ([7, 8], 150001, "bfloat16"),
    ([6], 300007, "float32"), ([5, 0, 12, 1], 131072, "float16")])
def test_matches_the_walk(new, V, dtype, tree, drawn):
    kept = [check(*case(new, V, dtype, tree, drawn, seed))[0].sum() for seed in range(3)]
    assert max(kept) > 0


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("tree", [False, True])
def test_ties_and_borders(tree, drawn):
    """Probabilities and numbers in few binary digits: tests and draws that
    fall on a border exactly, rejected mass that runs out."""
    for seed in range(12):
        check(*case([9, 5, 17], 40, "float32", tree, drawn, seed, sharp=2.0, grid=16))


def greedy_walk(p, tokens, starts, parents):
    p = np.asarray(p, np.float64)
    p = np.where(np.isnan(p), -np.inf, p)
    B, V = len(starts) - 1, p.shape[1]
    kept, path, nxt = np.zeros(B, int), np.full(p.shape[0], -1), np.full(B, -1)
    for b in range(B):
        s0, n = starts[b], min(starts[b + 1] - starts[b], 1024)
        if n <= 0:
            continue
        keep = [0]
        while True:
            best = int(p[s0 + keep[-1]].argmax())
            best = best if p[s0 + keep[-1]][best] > -np.inf else -1
            hit = [j for j in range(keep[-1] + 1, n) if (j - 1 if parents is None else parents[s0 + j]) == keep[-1]
                   and 0 <= tokens[s0 + j] < V and tokens[s0 + j] == best]
            if not hit:
                break
            keep.append(hit[0])
        kept[b], path[s0:s0 + len(keep)], nxt[b] = len(keep), keep, best
    return kept, path, nxt


def check_greedy(p, tokens, starts, parents):
    i32 = lambda x: None if x is None else torch.as_tensor(np.asarray(x, np.int32)).to(DEV)
    want = greedy_walk(p.double().cpu().numpy(), tokens, starts, parents)
    got = htree_amd.verify_drafts(p.to(DEV), torch.as_tensor(np.asarray(tokens, np.int64)).to(DEV), i32(starts),
                                  parents=i32(parents))
    for name, a, b in zip(got._fields, got, want):
        assert np.array_equal(a.cpu().numpy(), b), (name, a.cpu().numpy()[:20], b[:20])
    return want


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("new,V,dtype", [([6], 32000, "float32"), ([1, 0, 3], 1, "float32"), ([24] * 5, 7, "bfloat16"),
                                         ([9, 5], 8, "float16"), ([2, 9, 1, 30], 8192, "float16"), ([5, 5], 8193, "float32"),
                                         ([64, 65], 2047, "bfloat16"), ([3] * 300, 301, "bfloat16"), ([7, 8], 150001, "bfloat16"),
                                         ([1200], 40, "float32"),
                                         ([40, 1, 30], 1000003, "float32")])
def test_greedily(new, V, dtype, tree):
    """Scores of any size, equal ones among them, drafts half of which are what
    the target says."""
    kept = 0
    for seed in range(3):
        p, _, tokens, starts, parents, _, _ = case(new, V, dtype, tree, False, seed)
        g = np.random.default_rng(seed)
        scores = (torch.randn(p.shape, generator=torch.Generator().manual_seed(seed)) * 8).round() / 4
        scores = (scores * (10.0 ** 3 if seed else 1.0)).to(DT[dtype])
        best = scores.float().numpy().argmax(1)
        for b in range(len(new)):
            for j in range(1, new[b]):
                if g.random() < 0.5:
                    tokens[starts[b] + j] = best[starts[b] + (j - 1 if parents is None else parents[starts[b] + j])]
        if seed == 2:
            scores[g.random(p.shape) < 0.3] = float("nan")
            scores[::3] = scores[::3].clamp(max=0) - float("inf")
            scores[1::5, V // 2] = float("inf")
            if len(scores) > 1:
                scores[-1] = float("nan")
        kept = max(kept, check_greedy(scores, tokens, starts, parents)[0].max())
    assert kept > 1 or sum(new) < 20  # the larger cases accept something


def test_greedily_is_what_ones_and_zeros_give():
    p, _, tokens, starts, parents, u, d = case([20, 20, 20], 300, "float32", True, False, 3)
    one = torch.nn.functional.one_hot(p.argmax(1), 300).float()
    a = check_greedy(p, tokens, starts, parents)
    b = check(one, None, tokens, starts, parents, u, d)
    assert all(np.array_equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("drawn", [False, True])
def test_more_rows_than_are_looked_at(drawn):
    new, V = [1500, 3], 20
    p, q, tokens, starts, parents, u, d = case(new, V, "float32", False, drawn, 3)
    check(p, q, tokens, starts, parents, u * 0, d)  # a number of 0 accepts what has mass
    parents = np.concatenate([np.zeros(1500, int) - (np.arange(1500) == 0), [-1, 0, 1]])
    check(p, q, tokens, starts, parents, u * 0 + 0.999, d)


def test_one_row_of_everything():
    """A target equal to the drafter accepts everything; a token of no mass is
    never accepted; nothing left draws from the target itself."""
    V = 100
    p = torch.softmax(torch.randn(5, V, generator=torch.Generator().manual_seed(1)), -1)
    tokens, starts = [0, 3, 4, 5, 6], [0, 5]
    kept, path, nxt = check(p, p, tokens, starts, None, [0.999999] * 5, [0.5])
    assert kept[0] == 5
    p0 = p.clone()
    p0[0, 3] = 0
    assert check(p0, None, tokens, starts, None, [0.0] * 5, [0.5])[0][0] == 1
    one = torch.zeros(5, V)
    one[:, 7] = 0.5  # does not sum to one: rejected, and nothing else is there
    kept, _, nxt = check(one, None, [0, 7, 7, 7, 7], starts, None, [0.75] * 5, [0.9])
    assert kept[0] == 1 and nxt[0] == 7
    assert check(torch.zeros(5, V), None, tokens, starts, None, [0.0] * 5, [0.5])[2][0] == -1
    assert check(torch.zeros(5, V), p, tokens, starts, None, [0.0] * 5, [0.5])[2][0] == -1


def test_entries_that_are_no_probabilities():
    p, q, tokens, starts, parents, u, d = case([9, 9, 9], 300, "float32", True, True, 5)
    g = np.random.default_rng(2)
    for x in (p, q):
        at = torch.as_tensor(g.integers(0, 300, (27, 40)))
        bad = torch.tensor([float("nan"), float("inf"), -float("inf"), -1.0, torch.finfo(torch.float32).min])
        x.scatter_(1, at, bad[torch.as_tensor(g.integers(0, 5, (27, 40)))])
    check(p, q, tokens, starts, parents, u, d)
    check(p, None, tokens, starts, parents, u, d)
    check(torch.full_like(p, float("nan")), q, tokens, starts, parents, u, d)


def test_damaged_trees_tokens_and_numbers():
    for seed in range(6):
        p, q, tokens, starts, parents, u, d = case([20, 20, 20], 30, "float32", True, True, seed)
        g = np.random.default_rng(seed)
        parents[g.integers(0, 60, 8)] = g.integers(-5, 70, 8)
        tokens[g.integers(0, 60, 6)] = [-1, 30, 2 ** 40, -2 ** 40, 31, 2 ** 31]
        u[g.integers(0, 60, 6)] = [np.nan, -1, 1, 2, np.inf, 0]
        for last in ([np.nan, -3, 0], [1, 2, np.inf], [0.99999994, 1e-40, -0.0]):
            check(p, q, tokens, starts, parents, u, last)
            check(p, None, tokens, starts, parents, u, last)


def test_same_token_twice():
    """Siblings of one token: without a drafter's probabilities the second one
    finds nothing left."""
    p, q, tokens, starts, _, u, d = case([9], 50, "float32", False, True, 8)
    parents = np.array([-1] + [0] * 8)
    top = int(p[0].argmax())
    for q_ in (None, q):
        for u_ in (0.999, 0.3, 0.0):
            check(p, q_, [0] + [top] * 8, starts, parents, [u_] * 9, d)
            check(p, q_, [0, top, 3, top, 3, 3, 4, top, 4], starts, parents, [u_] * 9, d)


@pytest.mark.parametrize("dtype", list(DT))
def test_strides_and_offsets(dtype):
    """Rows that begin at any element, probabilities inside a larger tensor,
    rows behind the last request."""
    p, q, tokens, starts, parents, u, d = case([7, 5, 4], 1003, dtype, True, True, 4)
    starts = starts[:3]  # the last four rows are no request's
    d = d[:2]
    wide = torch.full((16, 2100), float("nan"), dtype=DT[dtype], device=DEV)
    wide[:, 3:1006], wide[:, 1017:2020] = p.to(DEV), q.to(DEV)
    check(wide[:, 3:1006], wide[:, 1017:2020], tokens, starts, parents, u, d)
    check(wide[:, 3:1006], None, tokens, starts, parents, u, d)


def test_past_32_bits():
    """Rows 2^30 entries apart: the last ones lie behind 2^32 of them."""
    p, q, tokens, starts, parents, u, d = case([3, 6], 1003, "bfloat16", True, True, 6)
    big = torch.empty(9, 1 << 30, dtype=torch.bfloat16, device=DEV)
    wide_p, wide_q = big[:, 5:1008], big[:, 1 << 29:(1 << 29) + 1003]
    wide_p.copy_(p), wide_q.copy_(q)
    check(wide_p, wide_q, tokens, starts, parents, u, d)
    check(wide_p, None, tokens, starts, parents, u, d)
    check_greedy(wide_p, tokens, starts, parents)


def test_starts_that_are_no_ranges_touch_nothing_outside():
    p, q, tokens, starts, parents, u, d = case([7, 5, 4], 100, "float32", True, True, 4)
    i32 = lambda x: torch.as_tensor(np.asarray(x, np.int32)).to(DEV)
    buf = torch.full((200,), -9, dtype=torch.int32, device=DEV)
    nxt = torch.full((60,), -9, dtype=torch.int64, device=DEV)
    out = htree_amd.Verified(buf[16:19], buf[64:80], nxt[20:23])
    f = lambda x: torch.as_tensor(np.asarray(x)).to(DEV)
    for bad in ([0, 50, 3, 16], [-4, 7, -2 ** 31, 2 ** 31 - 1], [16, 12, 5, 0], [3, 3, 3, 3]):
        for q_ in (q.to(DEV), None):
            htree_amd.verify_drafts(p.to(DEV), f(tokens), i32(bad), f(u), f(d), draft_probs=q_, parents=i32(parents),
                                    out=out)
    torch.cuda.synchronize()
    got = buf.cpu().numpy()
    assert (got[:16] == -9).all() and (got[19:64] == -9).all() and (got[80:] == -9).all()
    assert (nxt[:20] == -9).all() and (nxt[23:] == -9).all()


def test_nothing_to_verify():
    z = lambda *n, t=torch.float32: torch.zeros(n, dtype=t, device=DEV)
    v = htree_amd.verify_drafts(z(0, 9), z(0, t=torch.int64), z(3, t=torch.int32), z(0), z(2))
    assert v.kept.tolist() == [0, 0] and v.next_tokens.tolist() == [-1, -1] and v.path.numel() == 0
    v = htree_amd.verify_drafts(z(2, 9), z(2, t=torch.int64), z(1, t=torch.int32), z(2), z(0))
    assert v.kept.numel() == 0 and v.path.tolist() == [-1, -1]


def test_most_requests():
    g = np.random.default_rng(0)
    check(*case(list(g.integers(0, 4, 4096)), 33, "float32", True, True, 1))


@pytest.mark.parametrize("drawn", [False, True])
def test_what_is_kept_is_distributed_as_the_target(drawn):
    """4096 requests with one target, drafts of a quite different drafter: the
    token after the first one (accepted, or drawn) has the target's
    probabilities.  A count of N p differs by over 5 of its standard
    deviations with a chance of 6e-7 a token."""
    g = np.random.default_rng(11)
    N, V, n = 4096, 6, 4
    p0 = np.array([0.4, 0.05, 0.25, 0.1, 0.15, 0.05])
    q0 = np.array([0.1, 0.3, 0.05, 0.3, 0.05, 0.2])
    starts = np.arange(N + 1) * n
    parents = np.tile([-1, 0, 0, 0], N)  # three drafts of the first token
    tokens = g.choice(V, p=q0, size=N * n) if drawn else np.tile([0, 1, 3, 4], N)
    p, q = (torch.as_tensor(np.tile(x, (N * n, 1))) for x in (p0, q0))
    u, d = g.random(N * n, dtype=np.float32), g.random(N, dtype=np.float32)
    kept, path, nxt = check(p.float(), q.float() if drawn else None, tokens, starts, parents, u, d)
    then = np.where(kept > 1, tokens[starts[:-1] + path[starts[:-1] + np.minimum(kept - 1, n - 1)]], nxt)
    counts = np.bincount(then, minlength=V)
    assert np.all(np.abs(counts - N * p0) <= 5 * np.sqrt(N * p0 * (1 - p0))), counts


def test_refusals():
    f = lambda *n, t=torch.float32: torch.zeros(n, dtype=t, device=DEV)
    i32, i64 = torch.int32, torch.int64
    ok = dict(target_probs=f(3, 9), tokens=f(3, t=i64), starts=f(2, t=i32), uniforms=f(3), draws=f(1))
    htree_amd.verify_drafts(**ok)
    bad = [dict(target_probs=f(3, 9, t=torch.float64)), dict(target_probs=f(3, 9, 1)), dict(target_probs=f(3, 0)),
           dict(target_probs=f(9, 3).t()), dict(target_probs=f(4, 9)), dict(tokens=f(3, t=i32)), dict(tokens=f(2, t=i64)),
           dict(tokens=f(6, t=i64)[::2]), dict(starts=f(3, t=i32)), dict(starts=f(2, t=i64)),
           dict(uniforms=f(3, t=torch.float64)), dict(uniforms=f(4)), dict(draws=f(1, 1)), dict(draws=f(2)), dict(starts=f(4098, t=i32), draws=f(4097)), dict(uniforms=None), dict(draws=None),
           dict(uniforms=None, draws=None, draft_probs=f(3, 9)), dict(starts=f(0, t=i32)),
           dict(draft_probs=f(3, 8)), dict(draft_probs=f(3, 9, t=torch.bfloat16)), dict(parents=f(3, t=i64)),
           dict(parents=f(4, t=i32)), dict(tokens=torch.zeros(3, dtype=i64)), dict(draft_probs=torch.zeros(3, 9)),
           dict(out=htree_amd.Verified(f(2, t=i32), f(3, t=i32), f(1, t=i64))),
           dict(out=htree_amd.Verified(f(1, t=i32), f(3, t=i32), f(1, t=i32))),
           dict(out=htree_amd.Verified(f(1, t=i32), ok["starts"].expand(2)[:1].repeat(3)[:2], f(1, t=i64))),
           dict(out=htree_amd.Verified(ok["starts"][:1], f(3, t=i32), f(1, t=i64))),
           dict(out=htree_amd.Verified(f(1, t=i32), f(3, t=i32), ok["tokens"][1:2]))]
    both = f(3, t=i32)
    bad.append(dict(out=htree_amd.Verified(both[2:], both, f(1, t=i64))))
    for i, kw in enumerate(bad):
        with pytest.raises(AssertionError):
            htree_amd.verify_drafts(**dict(ok, **kw))
            print("not refused:", i)

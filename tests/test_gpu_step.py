"""The serving calls together, as a program runs them: a small model decodes
with drafted trees, token for token what it decodes without, requests are
forked on the way, and a step is captured."""
import numpy as np
import pytest
import torch

import htree_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
LAYERS, H, HKV, D, E, VOCAB, PAGE, PAGES, WIDTH = 2, 4, 2, 32, 64, 61, 16, 80, 12


def i32(x):
    return torch.as_tensor(np.asarray(x, np.int64)).to(torch.int32).to(DEV)


class Model:
    """Attention layers with normed heads, fp32."""

    def __init__(self, seed):
        g = torch.Generator().manual_seed(seed)
        rand = lambda *n: torch.randn(*n, generator=g).to(DEV)
        self.embed = rand(VOCAB, E)
        self.qkv = [rand(E, (H + 2 * HKV) * D) * E ** -0.5 for _ in range(LAYERS)]
        self.out = [rand(H * D, E) * (H * D) ** -0.5 for _ in range(LAYERS)]
        self.norm = [(1 + 0.1 * rand(D), 1 + 0.1 * rand(D)) for _ in range(LAYERS)]
        self.head = rand(E, VOCAB)
        self.cos, self.sin = htree_amd.rope_cache(D, 400, 10000.0, DEV)

    def step(self, tokens, t, kc, vc, table, parents):
        x = self.embed[tokens]
        for l in range(LAYERS):
            y = (x @ self.qkv[l]).view(-1, H + 2 * HKV, D)
            q, k = htree_amd.head_norm(y[:, :H], y[:, H:H + HKV], *self.norm[l], positions=t.positions, cos=self.cos,
                                       sin=self.sin)
            htree_amd.cache_append(k, y[:, H + HKV:], kc[l], vc[l], t.slots)
            o = htree_amd.draft_attention(q, kc[l], vc[l], table, t.lens, t.starts, parents=parents)
            x = x + o.reshape(-1, H * D) @ self.out[l]
        return x @ self.head

    def whole(self, tokens):
        """Scores after each token of a sequence, in 64 bits and without the framework."""
        n = len(tokens)
        x = self.embed.double()[torch.as_tensor(tokens).to(DEV)]
        c, s = self.cos[:n].double()[:, None], self.sin[:n].double()[:, None]
        mask = torch.full((n, n), -torch.inf, dtype=torch.float64, device=DEV).triu(1)
        for l in range(LAYERS):
            y = (x @ self.qkv[l].double()).view(n, H + 2 * HKV, D)

            def normed(z, w):
                z = z * (z.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w.double()
                a, b = z.chunk(2, -1)
                return torch.cat([a * c - b * s, b * c + a * s], -1)

            q, k = normed(y[:, :H], self.norm[l][0]), normed(y[:, H:H + HKV], self.norm[l][1])
            k, v = (z.repeat_interleave(H // HKV, 1).transpose(0, 1).contiguous() for z in (k, y[:, H + HKV:]))
            p = torch.softmax(q.transpose(0, 1) @ k.transpose(1, 2).contiguous() * D ** -0.5 + mask, -1)
            x = x + (p @ v).transpose(0, 1).reshape(n, H * D) @ self.out[l].double()
        return x @ self.head.double()

    def greedy(self, prompt, n):
        """The next n tokens, and how far ahead of the others each was at least."""
        seq, margin = list(prompt), np.inf
        for _ in range(n):
            top = self.whole(seq)[-1].topk(2)
            margin = min(margin, float(top.values[0] - top.values[1]))
            seq.append(int(top.indices[0]))
        return seq, margin


def drafts(seq, truth, n, g):
    """A tree of n tokens after the last of seq: its first row is that token,
    most branches follow what the model will say, others do not."""
    tokens, parents, depth = [seq[-1]], [-1], [0]
    for j in range(1, n):
        up = int(g.integers(max(0, j - 4), j))
        d = depth[up] + 1
        at = len(seq) - 1 + d
        good = at < len(truth) and g.random() < 0.6
        tokens.append(truth[at] if good else int(g.integers(0, VOCAB)))
        parents.append(up)
        depth.append(d)
    return tokens, parents


@pytest.mark.parametrize("layout", ["stacked", "list"])
def test_decoding_with_drafts(layout):
    """Greedy decoding with drafted trees of a prompt, its forks after a few
    steps, and another request: every token is the 64-bit model's own."""
    m, g = Model(3), np.random.default_rng(3)
    prompts = [list(g.integers(0, VOCAB, n)) for n in (19, 33)]
    if layout == "stacked":
        kc, vc = (torch.zeros(LAYERS, PAGES, PAGE, HKV, D, device=DEV) for _ in range(2))
    else:
        kc, vc = ([torch.zeros(PAGES, PAGE, HKV, D, device=DEV) for _ in range(LAYERS)] for _ in range(2))
    truth, margins = zip(*(m.greedy(p, 40) for p in prompts))
    assert min(margins) > 1e-4  # fp32 against 64 bits
    table = torch.full((2, WIDTH), -1, dtype=torch.int32, device=DEV)
    lens = i32([0, 0])
    free = htree_amd.unused_pages(table, lens, PAGE, PAGES).pages
    # the prompts but their last token, then trees
    n0 = [len(p) - 1 for p in prompts]
    t = htree_amd.page_tables(lens, i32(n0), table, free, PAGE, PAGES, sum(n0))
    m.step(torch.as_tensor(prompts[0][:-1] + prompts[1][:-1]).to(DEV), t, kc, vc, table, None)
    lens, seqs, most = t.lens, [list(p) for p in prompts], 0
    for step in range(9):
        if step == 4:  # three samples of the first request, the second beside them
            free = htree_amd.unused_pages(table, lens, PAGE, PAGES).pages
            f = htree_amd.fork_requests(table, lens, i32([0, 1, 0, 0]), free, PAGE, PAGES)
            htree_amd.copy_pages(kc, vc, f.copy_from, f.copy_to, f.copy_tokens)
            table, lens = f.block_table, f.lens
            seqs, truth = [list(seqs[i]) for i in (0, 1, 0, 0)], [truth[i] for i in (0, 1, 0, 0)]
            # one of them goes another way
            seqs[2][-1] = (seqs[2][-1] + 1) % VOCAB
            truth[2], margin = m.greedy(seqs[2], 30)
            assert margin > 1e-4
        if step == 7:  # the second request is done
            lens = lens * i32([1, 0, 1, 1])
        B = len(seqs)
        n = [int(x) for x in g.integers(1, 9, B)]
        if step >= 7:
            n[1] = 0
        trees = [drafts(s, w, k, g) if k else ([], []) for s, w, k in zip(seqs, truth, n)]
        tokens = torch.as_tensor(sum((a for a, _ in trees), [])).to(DEV)
        parents = i32(sum((b for _, b in trees), []))
        free = htree_amd.unused_pages(table, lens, PAGE, PAGES)
        t = htree_amd.page_tables(lens, i32(n), table, free.pages, PAGE, PAGES, sum(n), parents=parents)
        scores = m.step(tokens, t, kc, vc, table, parents)
        probs = torch.nn.functional.one_hot(scores.argmax(-1), VOCAB).float()
        v = htree_amd.verify_drafts(probs, tokens, t.starts, torch.rand(sum(n), device=DEV), torch.rand(B, device=DEV),
                                    parents=parents)
        greedy = htree_amd.verify_drafts(scores, tokens, t.starts, parents=parents)
        assert all(torch.equal(x, y) for x, y in zip(v, greedy))
        htree_amd.keep_drafts(kc, vc, t.slots, t.starts, v.path, v.kept)
        held = sum(-(-int(x) // PAGE) for x in lens + v.kept)
        lens = lens + v.kept
        kept, path, nxt, starts = v.kept.tolist(), v.path.tolist(), v.next_tokens.tolist(), t.starts.tolist()
        for b in range(B):
            if n[b] == 0:
                assert kept[b] == 0 and nxt[b] == -1
                continue
            seqs[b] += [int(tokens[starts[b] + i]) for i in path[starts[b] + 1:starts[b] + kept[b]]] + [nxt[b]]
            k = min(len(seqs[b]), len(truth[b]))
            assert seqs[b][:k] == truth[b][:k], (step, b)
            assert len(seqs[b]) - 1 == int(lens[b])
            most = max(most, kept[b])
        u = htree_amd.unused_pages(table, lens, PAGE, PAGES)
        if step < 4:
            assert int(u.count) == PAGES - held
    assert most > 3


def test_a_captured_step_with_drafts():
    """Pages, tables, norms, append, attention, verification, the move of what
    was kept and the next lengths in one graph that carries a batch on by
    itself, replayed against the same step run eagerly on its own state."""
    m, g = Model(5), np.random.default_rng(5)
    B, n = 3, 6
    rows = B * n

    class State:
        def __init__(self):
            self.kc, self.vc = (torch.zeros(LAYERS, PAGES, PAGE, HKV, D, device=DEV) for _ in range(2))
            self.table = torch.full((B, WIDTH), -1, dtype=torch.int32, device=DEV)
            self.lens = i32([0, 0, 0])

        def step(self, tokens, parents, u, d):
            new = i32_new
            free = htree_amd.unused_pages(self.table, self.lens, PAGE, PAGES).pages
            t = htree_amd.page_tables(self.lens, new, self.table, free, PAGE, PAGES, rows, parents=parents)
            probs = torch.softmax(m.step(tokens, t, self.kc, self.vc, self.table, parents), -1)
            v = htree_amd.verify_drafts(probs, tokens, t.starts, u, d, parents=parents)
            htree_amd.keep_drafts(self.kc, self.vc, t.slots, t.starts, v.path, v.kept)
            self.lens.add_(v.kept)
            return v

    i32_new = i32([n] * B)
    tokens = torch.zeros(rows, dtype=torch.int64, device=DEV)
    parents, u, d = i32([-1] * rows), torch.zeros(rows, device=DEV), torch.zeros(B, device=DEV)
    a, b = State(), State()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        State().step(tokens, parents, u, d)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = a.step(tokens, parents, u, d)
    a.lens.zero_()
    moved = 0
    for rep in range(8):
        tokens.copy_(torch.as_tensor(g.integers(0, VOCAB, rows)))
        parents.copy_(i32(np.concatenate([[-1] + [int(g.integers(0, j)) for j in range(1, n)] for _ in range(B)])))
        u.copy_(torch.as_tensor(g.random(rows, dtype=np.float32)) * 0.1)
        d.copy_(torch.as_tensor(g.random(B, dtype=np.float32)))
        graph.replay()
        torch.cuda.synchronize()
        want = b.step(tokens, parents, u, d)
        for x, y in zip(got, want):
            assert torch.equal(x, y), rep
        assert torch.equal(a.lens, b.lens) and torch.equal(a.table, b.table)
        live = torch.arange(WIDTH * PAGE, device=DEV) < a.lens[:, None]
        at = a.table.repeat_interleave(PAGE, 1).long() * PAGE + torch.arange(WIDTH * PAGE, device=DEV) % PAGE
        for x, y in ((a.kc, b.kc), (a.vc, b.vc)):
            assert torch.equal(x.flatten(1, 2)[:, at[live]], y.flatten(1, 2)[:, at[live]])
        moved = max(moved, int(got.kept.max()))
    assert moved > 1


def test_on_another_stream():
    """All calls on a side stream, its work ordered by events alone."""
    side = torch.cuda.Stream()
    big = torch.randn(4096, 4096, device=DEV)
    kc, vc = (torch.randn(3, PAGES, PAGE, HKV, D, device=DEV) for _ in range(2))
    want_k = kc.clone()
    want_k[:, 7, :5] = kc[:, 3, :5]
    p = torch.softmax(torch.randn(6, 50000, device=DEV), -1)
    toks, starts = torch.arange(6, device=DEV), i32([0, 6])
    u, d = torch.full((6,), 0.99, device=DEV), torch.full((1,), 0.5, device=DEV)
    x, w = torch.randn(64, 4, 64, device=DEV), torch.randn(64, device=DEV)
    torch.cuda.synchronize()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            big = big @ big * 1e-3
        late = big[0, 0] * 0  # what follows has to wait for the products
        frm = (i32([3]) + late.int())
        htree_amd.copy_pages(kc, vc, frm, i32([7]), i32([5]))
        v = htree_amd.verify_drafts(p + late, toks, starts, u, d)
        used = htree_amd.unused_pages((i32([[1, 2]]) + late.int()), i32([32]), PAGE, PAGES)
        y = htree_amd.head_norm(x + late, x + late, w, w)[0]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(kc, want_k) and int(used.count) == PAGES - 2
    assert v.kept.tolist() == [1] and 0 <= int(v.next_tokens) < 50000
    r = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
    assert float((y - r).abs().max()) < 1e-4


def test_two_streams_at_once():
    """Calls that overlap, each with workspaces of its own: what they give is
    what they give one after another."""
    g = torch.Generator(device=DEV).manual_seed(9)
    jobs = []
    for i in range(2):
        p, q = (torch.softmax(4 * torch.randn(24, 140001, generator=g, device=DEV), -1) for _ in range(2))
        toks = torch.randint(140001, (24,), generator=g, device=DEV)
        u, d = torch.rand(24, generator=g, device=DEV), torch.rand(4, generator=g, device=DEV)
        table = torch.randint(300000, (600, 900), generator=g, device=DEV).int()
        lens = torch.randint(900 * PAGE, (600,), generator=g, device=DEV).int()
        x = [torch.randn(3000, h, 128, generator=g, device=DEV).bfloat16().requires_grad_() for h in (16, 2)]
        w = [torch.randn(128, generator=g, device=DEV).requires_grad_() for _ in range(2)]
        dy = [torch.randn(3000, h, 128, generator=g, device=DEV).bfloat16() for h in (16, 2)]
        jobs.append((p, q, toks, u, d, table, lens, x, w, dy))

    def run(p, q, toks, u, d, table, lens, x, w, dy):
        out = [*htree_amd.verify_drafts(p, toks, i32([0, 6, 12, 18, 24]), u, d, draft_probs=q),
               *htree_amd.verify_drafts(p, toks, i32([0, 6, 12, 18, 24])), *htree_amd.unused_pages(table, lens, PAGE, 300000)]
        y = htree_amd.head_norm(*x, *w)
        return out + [*y, *torch.autograd.grad(y, [*x, *w], dy)]

    want = [run(*j) for j in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for _ in range(4):
        got = []
        for s, j in zip(streams, jobs):
            with torch.cuda.stream(s):
                got.append([run(*j) for _ in range(3)])
        torch.cuda.synchronize()
        for runs, y in zip(got, want):
            for r in runs:
                assert all(torch.equal(a, b) for a, b in zip(r, y))

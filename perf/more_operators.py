"""What surrounds attention in a serving step, as measured cases: drafted
tokens verified against the target's probabilities, accepted ones moved
together in the paged cache, requests forked, pages found that none holds,
and queries and keys normed by head and rotated, which training needs too.

A pass is one operator.  Where `own` is false it is computed in plain torch
operations, where it is true by htree_amd's entry points.

New tokens of all requests are packed: rows starts[b] .. starts[b + 1] - 1 are
request b's.  Its first row is the token its last step decided on, the others
are drafts; parents[row] is the index, among its request's rows, of the token
it was drafted after (without parents: the row before).  The cache holds all
layers, [layers, pages, page, H_kv, D]; a slot is page * page_size + offset.
"""
import math
import random

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


# ------------------------------------------------------------------ cases
def _verify(name, B, new, V, dtype, tree, drawn):
    return dict(name=name, op="verify", B=B, new=new, V=V, dtype=dtype, tree=tree, drawn=drawn)


def _keep(name, B, new, layers, Hkv, D, dtype, page):
    return dict(name=name, op="keep", B=B, new=new, layers=layers, Hkv=Hkv, D=D, dtype=dtype, page=page)


def _fork(name, B, fan, ctx, layers, Hkv, D, dtype, page):
    return dict(name=name, op="fork", B=B, fan=fan, ctx=ctx, layers=layers, Hkv=Hkv, D=D, dtype=dtype,
                page=page)


def _unused(name, B, ctx, page, spare, held):
    return dict(name=name, op="unused", B=B, ctx=ctx, page=page, spare=spare, held=held)


def _norm(name, rows, H, Hkv, D, dtype, rope, train):
    return dict(name=name, op="norm", rows=rows, H=H, Hkv=Hkv, D=D, dtype=dtype, rope=rope, train=train)


def listed():
    """new, ctx are the longest request's; the others are ragged below."""
    return [
        # one request's chain of five drafts: latency
        _verify("verify_1x5", 1, 6, 32000, "float32", False, True),
        # a batch's chains with both models' probabilities in 16 bits
        _verify("verify_64x8", 64, 9, 128000, "bfloat16", False, True),
        # fixed trees of up to 24 tokens for each of a full batch
        _verify("verify_256_trees", 256, 24, 32768, "float32", True, False),
        # trees drawn from the drafter, an odd vocabulary
        _verify("verify_16_drawn_trees", 16, 24, 50001, "float32", True, True),
        # accepted drafts of a small batch, one layer's cache
        _keep("keep_16", 16, 24, 1, 2, 128, "bfloat16", 16),
        # of a full batch, all layers
        _keep("keep_256x32", 256, 64, 32, 8, 128, "bfloat16", 16),
        # eight samples of one prompt
        _fork("fork_1x8", 1, 8, 4001, 16, 4, 32, "float32", 64),
        # beams of 64 prompts reordered
        _fork("fork_beams_256", 256, 1, 395, 16, 4, 128, "bfloat16", 16),
        # a batch's pages after a step
        _unused("unused_64", 64, 16384, 16, 5000, 0),
        # a large pool of many requests, some pages held for others
        _unused("unused_1024", 1024, 32768, 16, 100003, 20000),
        # a decoding step's queries and keys, rotated: latency
        _norm("norm_step_64", 64, 32, 2, 128, "bfloat16", True, False),
        # four training sequences of 16384, forward and backward
        _norm("norm_train_64k", 65536, 32, 4, 128, "bfloat16", False, True),
    ]


def _log(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))


def draw(rng):
    """A further case of the same ranges: one request to a full batch, small
    vocabularies to large, one layer to many, every type, odd sizes."""
    top = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["verify", "verify", "keep", "fork", "unused", "norm", "norm"])
        page = rng.choice([16, 16, 32, 64])
        dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
        H, Hkv, D = rng.choice([(32, 2, 128), (32, 4, 128), (64, 8, 128), (64, 4, 32), (8, 1, 128), (8, 2, 64),
                                (16, 4, 32), (4, 1, 64), (6, 2, 96), (16, 2, 256), (4, 4, 128)])
        if op == "verify":
            tree = rng.random() < 0.6
            c = _verify("", _log(rng, 1, 256), _log(rng, 2, 48), _log(rng, 1000, 160000),
                        rng.choice(["bfloat16", "float16", "float32", "float32"]), tree,
                        rng.random() < (0.4 if tree else 0.9))
            if c["B"] * c["new"] * c["V"] > 2 ** (26 if tree and c["drawn"] else 28):
                continue
        elif op == "keep":
            c = _keep("", _log(rng, 1, 256), _log(rng, 2, 64), _log(rng, 1, 40), Hkv, D, dtype, page)
            if _pool(c) * page * c["layers"] * Hkv * D > 2 ** 30:
                continue
        elif op == "fork":
            c = _fork("", _log(rng, 1, 256), rng.choice([1, 2, 3, 8]), _log(rng, 1, 8192), _log(rng, 1, 40),
                      Hkv, D, dtype, page)
            if c["B"] * c["fan"] > 512 or _pool(c) * page * c["layers"] * Hkv * D > 2 ** 29:
                continue
        elif op == "unused":
            c = _unused("", _log(rng, 1, 1024), _log(rng, 1, 65536), page, _log(rng, 1, 100000),
                        rng.choice([0, _log(rng, 1, 20000)]))
        else:
            train = rng.random() < 0.5
            c = _norm("", _log(rng, 1, 65536), H, Hkv, D, dtype, not train or rng.random() < 0.3, train)
        if _cost(c) <= top:
            del c["name"]
            return c


def _ragged(c, what, least):
    """A length for each request, the longest (the case's own) first."""
    r = random.Random("%s %s %s %s" % (what, c["op"], c["B"], c[what]))
    return [c[what]] + [r.randint(min(least, c[what]), c[what]) for _ in range(c["B"] - 1)]


def _sources(c):
    """Which request each new one carries on from: `fan` of each, or the beams
    of groups of four reordered."""
    if c["fan"] > 1:
        return [i // c["fan"] for i in range(c["B"] * c["fan"])]
    r = random.Random("beams %s" % c["B"])
    return [r.randrange(i // 4 * 4, min(i // 4 * 4 + 4, c["B"])) for i in range(c["B"])]


def _pages(c):
    """Pages that each request holds (keep: at most a page for each side of
    its new tokens, which are all that its cases keep)."""
    if c["op"] == "keep":
        return [-(-(n + 5) // c["page"]) for n in _ragged(c, "new", 1)]
    return [-(-n // c["page"]) for n in _ragged(c, "ctx", c["ctx"] // 4)]


def _pool(c):
    return sum(_pages(c)) + (c["spare"] if c["op"] == "unused" else c["B"] * c.get("fan", 0) + 3)


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


def work(case):
    """Each input read once, each output written once: of the probabilities
    the rows that the next tokens are drawn from, of a table the live entries,
    of a cache the tokens that move."""
    c = case
    if c["op"] == "norm":
        e = 4 if c["dtype"] == "float32" else 2
        n = c["rows"] * (c["H"] + c["Hkv"]) * c["D"]
        b = (5 if c["train"] else 2) * n * e + (4 * c["rows"] + 4 * c["D"] * c["rows"] if c["rope"] else 0)
        return {"bytes": b, "flops": (20 if c["train"] else 8) * n}
    if c["op"] == "verify":
        e = 4 if c["dtype"] == "float32" else 2
        rows = sum(_ragged(c, "new", 2))
        both = 2 if c["drawn"] else 1
        # tokens, uniforms, parents in and the path out, an element of each row
        b = c["B"] * (c["V"] * e * both + 20) + rows * (16 + 4 * c["tree"] + e * both)
        return {"bytes": b, "flops": 2 * c["B"] * c["V"] * both}
    if c["op"] == "unused":
        live = sum(_pages(c))
        return {"bytes": 4 * (live + c["B"] + c["held"] + _pool(c)), "flops": live + _pool(c)}
    token = c["layers"] * c["Hkv"] * c["D"] * 2 * (4 if c["dtype"] == "float32" else 2)
    if c["op"] == "keep":
        moved = sum(_kept(n) - 1 for n in _ragged(c, "new", 1))
        return {"bytes": 2 * moved * token + 12 * sum(_ragged(c, "new", 1)), "flops": moved}
    ctx, pages, src = _ragged(c, "ctx", c["ctx"] // 4), _pages(c), _sources(c)
    copied = sum(ctx[s] % c["page"] for i, s in enumerate(src) if s in src[:i])
    entries = sum(pages[s] for s in src)
    return {"bytes": 2 * copied * token + 4 * (entries + len(src) * (max(pages) + 6)), "flops": entries}


def _kept(n):
    """How many of n new tokens the measured steps keep: the first and about
    a draft for each doubling of the tree."""
    return min(n, 1 + n.bit_length() // 2)


# ----------------------------------------------------------------- inputs
def _starts(new):
    s = torch.zeros(len(new) + 1, dtype=torch.int32, device="cuda")
    s[1:] = torch.tensor(new, device="cuda").cumsum(0)
    return s


def _rows(new, starts):
    """Of each row its request and its index there."""
    n = torch.tensor(new, device="cuda")
    r = torch.arange(len(new), device="cuda").repeat_interleave(n, output_size=sum(new))
    return r, torch.arange(sum(new), device="cuda") - starts[r].long()


def _siblings(parents, starts, r, most):
    """[rows, most] true where the row at that index of the same request is an
    earlier child of the same token."""
    at = (starts[r].long()[:, None] + torch.arange(most, device="cuda")).clamp(max=parents.numel() - 1)
    j = torch.arange(parents.numel(), device="cuda")[:, None]
    return (at < j) & (at >= starts[r].long()[:, None]) & (parents[at] == parents[:, None]), at


def _prepare_verify(c, seed, g):
    new = _ragged(c, "new", 2)
    starts, rows, V, t = _starts(new), sum(new), c["V"], DTYPES[c["dtype"]]
    r, j = _rows(new, starts)
    if c["tree"]:
        back = 1 + (torch.rand(rows, generator=g, device="cuda") ** 2 * torch.clamp(0.5 * j, 2, 8)).long()
        parents = torch.where(j == 0, -1, torch.clamp(j - back, min=0)).int()
    else:
        parents = (j - 1).int()
    same, _ = _siblings(parents, starts, r, max(new))
    rank = same.sum(1)
    logits = torch.randn(rows, V, generator=g, device="cuda") * 4
    p = torch.softmax(logits, -1)
    logits += torch.randn(rows, V, generator=g, device="cuda") * 0.7
    q = torch.softmax(logits, -1)
    after = (starts[r].long() + parents).clamp(min=0)
    if c["drawn"]:  # each draft drawn from the drafter's probabilities
        u = torch.rand(rows, 1, generator=g, device="cuda", dtype=torch.float64)
        tokens = torch.searchsorted(q.double().cumsum(1)[after], u).squeeze(1).clamp(max=V - 1)
    else:           # siblings are the drafter's likeliest
        top = logits.topk(min(V, int(rank.max()) + 1), -1).indices
        tokens = top[after, rank]
    return dict(p=p.to(t), q=q.to(t) if c["drawn"] else None, tokens=tokens.long().contiguous(), starts=starts,
                parents=parents if c["tree"] else None, ranks=int(rank.max()) + 1, most=max(new),
                uniforms=torch.rand(rows, generator=g, device="cuda"),
                draws=torch.rand(c["B"], generator=g, device="cuda"))


def _table(c, total, g):
    """Block table over a shuffled pool and the pool's other pages."""
    had = torch.tensor(_pages(c), device="cuda")
    pool = torch.randperm(total, generator=g, device="cuda").int()
    j = torch.arange(max(_pages(c)), device="cuda")
    at = (had.cumsum(0) - had)[:, None] + j
    return torch.where(j < had[:, None], pool[at.clamp(max=total - 1)], -1).int().contiguous(), pool[int(had.sum()):].contiguous()


def _caches(c, total, g):
    t = DTYPES[c["dtype"]]
    return [torch.randn(c["layers"], total, c["page"], c["Hkv"], c["D"], generator=g, device="cuda", dtype=t)
            for _ in range(2)]


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(op=c["op"])
    if c["op"] == "verify":
        s.update(_prepare_verify(c, seed, g))
        return s
    if c["op"] == "norm":
        t, H, Hkv, D = DTYPES[c["dtype"]], c["H"], c["Hkv"], c["D"]
        rand = lambda *n: torch.randn(*n, generator=g, device="cuda", dtype=t)
        if c["train"]:
            q, k = rand(c["rows"], H, D), rand(c["rows"], Hkv, D)
            s.update(gq=rand(c["rows"], H, D), gk=rand(c["rows"], Hkv, D))
        else:  # the rows of a fused projection
            qkv = rand(c["rows"], H + 2 * Hkv, D) * 2
            q, k = qkv[:, :H], qkv[:, H:H + Hkv]
        s.update(q=q, k=k, wq=1 + 0.1 * rand(D), wk=1 + 0.1 * rand(D), eps=1e-6, train=c["train"],
                 pos=None, cos=None, sin=None)
        if c["train"]:
            for x in ("q", "k", "wq", "wk"):
                s[x].requires_grad_()
        if c["rope"]:
            n = max(c["rows"], 1024)
            a = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] \
                * 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
            s.update(cos=a.cos().float(), sin=a.sin().float(),
                     pos=torch.randint(n, (c["rows"],), generator=g, device="cuda").int())
        return s
    page, total = c["page"], _pool(c)
    s.update(page=page, pages=total)
    table, free = _table(c, total, g)
    if c["op"] == "unused":
        # requests in groups of four share what they were forked from
        lead = torch.arange(c["B"], device="cuda") // 4 * 4
        shared = torch.tensor(_pages(c), device="cuda")
        shared = torch.minimum(shared, shared[lead]) // 3
        j = torch.arange(table.shape[1], device="cuda")
        s.update(table=torch.where(j < shared[:, None], table[lead], table).contiguous(),
                 lens=torch.tensor(_ragged(c, "ctx", c["ctx"] // 4), device="cuda").int(),
                 held=free[torch.randint(free.numel(), (c["held"],), generator=g, device="cuda")] if c["held"] else None)
        return s
    s["k"], s["v"] = _caches(c, total, g)
    if c["op"] == "keep":
        new = _ragged(c, "new", 1)
        starts = _starts(new)
        r, j = _rows(new, starts)
        at = j + torch.randint(5, (c["B"],), generator=g, device="cuda")[r]
        kept = torch.tensor([_kept(n) for n in new], device="cuda")
        # the first row and some of the others, in order: those of the least numbers
        key = torch.rand(sum(new), generator=g, device="cuda", dtype=torch.float64) - (j == 0).double()
        place = torch.empty_like(r)
        place[(key + 4 * r).sort(stable=True).indices] = torch.arange(sum(new), device="cuda")
        chosen = place - starts[r].long() < kept[r]
        to = starts[r].long() + chosen.long().cumsum(0) - 1 - (kept.cumsum(0) - kept)[r]
        path = torch.full((sum(new) + 1,), -1, dtype=torch.int32, device="cuda")
        path[torch.where(chosen, to, sum(new))] = j.int()
        path = path[:-1].clone()
        s.update(slots=table[r, at // page].long() * page + at % page, starts=starts, path=path, kept=kept.int())
    else:
        s.update(table=table, free=free, source=torch.tensor(_sources(c), device="cuda").int(),
                 lens=torch.tensor(_ragged(c, "ctx", c["ctx"] // 4), device="cuda").int())
    return s


# ------------------------------------------------------------- plain forms
def _verify_plain(s):
    """Every draft's test at once, in 64 bits: a sum in 32 bits would move the
    borders between tokens."""
    p, q, tokens, starts, n = s["p"], s["q"], s["tokens"], s["starts"].long(), s["most"]
    dev, rows, (B, V) = p.device, p.shape[0], (starts.numel() - 1, p.shape[1])
    r = torch.searchsorted(starts[1:].contiguous(), torch.arange(rows, device=dev), right=True)
    j = torch.arange(rows, device=dev) - starts[r]
    parents = (j - 1).int() if s["parents"] is None else s["parents"]
    same, at = _siblings(parents, starts, r, n)
    rank = same.sum(1)
    draft = j > 0
    after = (starts[r] + parents).clamp(min=0)
    u, px = s["uniforms"].double(), p[after, tokens].double()
    if q is None:
        seen = (same & (tokens[at] == tokens[:, None])).any(1)
        px = torch.where(seen, 0, px)
        passed = draft & (u * (1 - (same * px[at]).sum(1)) < px)
    else:
        qx = q[after, tokens].double()
        # of each row the multiple of q taken off, and what is left of p's mass
        off, left = torch.zeros(rows, device=dev, dtype=torch.float64), torch.ones(rows, device=dev, dtype=torch.float64)
        children = torch.zeros(rows, device=dev, dtype=torch.long).index_add_(0, after, draft.long())
        passed = torch.zeros_like(draft)
        for m in range(s["ranks"]):
            mine = draft & (rank == m)
            passed |= mine & (u * left[after] * qx < px - off[after] * qx)
            off = torch.where(children > m, off + left, off)
            if m + 1 < s["ranks"]:
                left = (p.double() - off[:, None] * q.double()).clamp_(min=0).sum(1)
    passed &= ~(same & passed[at]).any(1)
    # kept: every token on the way to the first row passed
    blocked = draft & ~passed
    j2 = torch.arange(n, device=dev)
    row = (starts[:-1, None] + j2).clamp(max=rows - 1)
    there = j2 < starts.diff()[:, None]
    up = torch.where(there, parents[row], -1)
    reach = (up[:, :, None] == j2).float() + torch.eye(n, device=dev)
    for _ in range(max(1, (n - 1).bit_length())):
        reach = torch.matmul(reach, reach).clamp(max=1.0)
    bad = (blocked[row] & there).float()
    keep = there & (torch.matmul(reach, bad[:, :, None]).squeeze(2) < 0.5)
    kept = keep.sum(1)
    path = torch.full((rows + 1,), -1, dtype=torch.int32, device=dev)
    path[torch.where(keep, starts[:-1, None] + keep.long().cumsum(1) - 1, rows)] = j2.int().expand(B, n)
    last = starts[:-1] + torch.where(keep, j2, 0).amax(1)
    left = p[last].double()
    if q is None:
        child = draft & (after == last[r])
        out = torch.zeros(B, V + 1, device=dev, dtype=torch.bool)
        out[r, torch.where(child, tokens, V)] = True
        left = torch.where(out[:, :V], 0, left)
    else:
        left = (left - off[last][:, None] * q[last].double()).clamp(min=0)
    left = torch.where((left.sum(1) > 0)[:, None], left, p[last].double())
    total = left.cumsum(1)
    end = torch.where(left > 0, torch.arange(V, device=dev), 0).amax(1)
    t = s["draws"].double() * total[:, -1]
    token = torch.minimum(torch.searchsorted(total, t[:, None], right=True).squeeze(1), end)
    return {"kept": kept.int(), "path": path[:rows], "next_tokens": token}


def _keep_plain(s):
    rows = s["slots"].numel()
    starts = s["starts"].long()
    row = torch.arange(rows, device=s["slots"].device)
    r = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    src = torch.where(row - starts[r] < s["kept"][r], starts[r] + s["path"], row)  # the others stay
    for x in (s["k"], s["v"]):
        flat = x.flatten(1, 2)
        flat[:, s["slots"]] = flat[:, s["slots"][src]]
    return {"k": s["k"], "v": s["v"]}


def _fork_plain(s):
    src, page, W = s["source"].long(), s["page"], s["table"].shape[1]
    dev, N = src.device, src.numel()
    lens = s["lens"][src]
    i = torch.arange(N, device=dev)
    first = torch.full((s["lens"].numel(),), N, device=dev).scatter_reduce_(0, src, i, "amin")
    copy = (lens % page > 0) & (first[src] != i)
    fresh = s["free"][(copy.long().cumsum(0) - 1).clamp(min=0)]
    j = torch.arange(W, device=dev)
    table = torch.where(j < ((lens + page - 1) // page)[:, None], s["table"][src], -1)
    at = (lens // page).clamp(max=W - 1).long()
    old = table[i, at]
    table[i, at] = torch.where(copy, fresh, old)
    a, b, n = torch.where(copy, old, -1), torch.where(copy, fresh, -1), torch.where(copy, lens % page, 0)
    # what does not move is written to itself: the first request's first token
    o = torch.arange(page, device=dev)
    moves = o < n[:, None]
    here = s["table"][0, 0].long() * page
    to = torch.where(moves, b.long()[:, None] * page + o, here).flatten()
    frm = torch.where(moves, a.long()[:, None] * page + o, here).flatten()
    for x in (s["k"], s["v"]):
        flat = x.flatten(1, 2)
        flat[:, to] = flat[:, frm]
    return {"table": table, "lens": lens, "copy_from": a, "copy_to": b, "copy_tokens": n,
            "pages_used": copy.sum().int().reshape(1), "k": s["k"], "v": s["v"]}


def _unused_plain(s):
    page, P = s["page"], s["pages"]
    live = torch.arange(s["table"].shape[1], device="cuda") < ((s["lens"] + page - 1) // page)[:, None]
    used = torch.zeros(P + 1, dtype=torch.bool, device="cuda")
    used[torch.where(live, s["table"], P).long().flatten()] = True
    if s["held"] is not None:
        used[s["held"].long()] = True
    free = ~used[:P]
    at = free.long().cumsum(0)
    pages = torch.full((P + 1,), -1, dtype=torch.int32, device="cuda")
    pages[torch.where(free, at - 1, P)] = torch.arange(P, device="cuda", dtype=torch.int32)
    return {"pages": pages[:P], "count": at[-1:].int()}


def _turn(x, cos, sin):
    if cos is None:
        return x
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _norm_plain(s):
    cos = sin = back = None
    if s["cos"] is not None:
        cos, sin = s["cos"][s["pos"].long()][:, None], s["sin"][s["pos"].long()][:, None]
        back = -sin
    out = {}
    for n, w in (("q", "wq"), ("k", "wk")):
        x, weight = s[n].detach().float(), s[w].detach().float()
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + s["eps"])
        out[n] = _turn(x * r * weight, cos, sin).to(s[n].dtype)
        if s["train"]:
            g = _turn(s["g" + n].float(), cos, back)
            out["d" + w] = (g * x * r).sum((0, 1)).to(s[w].dtype)
            g = g * weight
            out["d" + n] = (r * (g - x * r.square() * (g * x).mean(-1, keepdim=True))).to(s[n].dtype)
    return out


# -------------------------------------------------------------------- run
def run(state):
    s = state
    if own:
        import htree_amd

        if s["op"] == "verify":
            return htree_amd.verify_drafts(s["p"], s["tokens"], s["starts"], s["uniforms"], s["draws"],
                                           draft_probs=s["q"], parents=s["parents"])._asdict()
        if s["op"] == "keep":
            htree_amd.keep_drafts(s["k"], s["v"], s["slots"], s["starts"], s["path"], s["kept"])
            return {"k": s["k"], "v": s["v"]}
        if s["op"] == "fork":
            f = htree_amd.fork_requests(s["table"], s["lens"], s["source"], s["free"], s["page"], s["pages"])
            htree_amd.copy_pages(s["k"], s["v"], f.copy_from, f.copy_to, f.copy_tokens)
            return {"table": f.block_table, "lens": f.lens, "copy_from": f.copy_from, "copy_to": f.copy_to,
                    "copy_tokens": f.copy_tokens, "pages_used": f.pages_used, "k": s["k"], "v": s["v"]}
        if s["op"] == "unused":
            return htree_amd.unused_pages(s["table"], s["lens"], s["page"], s["pages"], held=s["held"])._asdict()
        q, k = htree_amd.head_norm(s["q"], s["k"], s["wq"], s["wk"], eps=s["eps"], positions=s["pos"],
                                   cos=s["cos"], sin=s["sin"])
        if not s["train"]:
            return {"q": q, "k": k}
        dq, dk, dwq, dwk = torch.autograd.grad((q, k), (s["q"], s["k"], s["wq"], s["wk"]), (s["gq"], s["gk"]))
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    return {"verify": _verify_plain, "keep": _keep_plain, "fork": _fork_plain, "unused": _unused_plain,
            "norm": _norm_plain}[s["op"]](s)


# ------------------------------------------------------------------ exact
def exact(case, seed):
    """The definition in 64 bits.  Verification and free pages are whole
    numbers alone."""
    c = case
    if c["op"] in ("verify", "unused"):
        return None
    s = prepare(case, seed)
    if c["op"] == "norm":
        return _norm_exact(s)
    # what is copied keeps its values: token by token, each read before any is written
    moves = []
    if c["op"] == "keep":
        starts, kept, path, slots = (s[n].tolist() for n in ("starts", "kept", "path", "slots"))
        for b in range(c["B"]):
            moves += [(slots[starts[b] + path[starts[b] + i]], slots[starts[b] + i]) for i in range(kept[b])]
    else:
        ctx, page, free = _ragged(c, "ctx", c["ctx"] // 4), c["page"], s["free"].tolist()
        table, had = s["table"].tolist(), set()
        for b in _sources(c):
            if b in had and ctx[b] % page:
                a, to = table[b][ctx[b] // page], free.pop(0)
                moves += [(a * page + i, to * page + i) for i in range(ctx[b] % page)]
            had.add(b)
    out = {}
    for n in ("k", "v"):
        flat = s[n].double().flatten(1, 2)
        if moves:
            a, b = torch.tensor(moves, device="cuda").t()
            flat.index_copy_(1, b, flat.index_select(1, a))
        out[n] = flat.view(s[n].shape)
    if c["op"] == "fork":
        out.update({n: None for n in ("table", "lens", "copy_from", "copy_to", "copy_tokens", "pages_used")})
    return out


def _norm_exact(s):
    """By complex numbers, and the gradient as the projection it is: what a
    normed vector can change by is what stands across it."""
    out = {}
    turn = None
    if s["cos"] is not None:
        at = s["pos"].long()
        turn = torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None]

    def turned(x, by):
        if by is None:
            return x
        h = x.shape[-1] // 2
        z = torch.complex(x[..., :h].contiguous(), x[..., h:].contiguous()) * by
        return torch.cat([z.real, z.imag], -1)

    for n, w in (("q", "wq"), ("k", "wk")):
        x, weight = s[n].detach().double(), s[w].detach().double()
        size = (torch.linalg.vector_norm(x, dim=-1, keepdim=True).square() / x.shape[-1] + s["eps"]).sqrt()
        unit = x / size
        out[n] = turned(unit * weight, turn)
        if s["train"]:
            g = turned(s["g" + n].double(), None if turn is None else turn.conj())
            out["d" + w] = (g * unit).sum((0, 1))
            g = g * weight
            out["d" + n] = (g - unit * (g * unit).sum(-1, keepdim=True) / x.shape[-1]) / size
    return out

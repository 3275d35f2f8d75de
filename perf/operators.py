"""Serving from a paged key/value cache, as measured cases: block tables and
slot maps from request lengths, keys and values rotated and appended to the
cache, and the attention of drafted tokens (or single ones, or a chunk of a
prompt) over it.

A pass is one call of an operator.  Where `own` is false it is computed in
plain torch operations, where it is true by htree_amd's entry points.

The cache is k_cache [pages, page, H_kv, D], v_cache the same; token p of
request b sits in page block_table[b, p // page] at offset p % page; a slot is
page * page_size + offset.  New tokens of all requests are packed: rows
starts[b] .. starts[b + 1] - 1 are request b's.  parents[row] is the index,
among its request's new tokens, of the token it was drafted after (-1: the
last cached one); without parents each follows the one before it.
"""
import math
import random

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


# ------------------------------------------------------------------ cases
def _tables(name, B, ctx, new, page, tree):
    return dict(name=name, op="tables", B=B, ctx=ctx, new=new, page=page, tree=tree)


def _append(name, B, ctx, new, H, Hkv, D, dtype, page, rope):
    return dict(name=name, op="append", B=B, ctx=ctx, new=new, H=H, Hkv=Hkv, D=D, dtype=dtype,
                page=page, rope=rope)


def _attend(name, B, ctx, new, H, Hkv, D, dtype, page, tree):
    return dict(name=name, op="attend", B=B, ctx=ctx, new=new, H=H, Hkv=Hkv, D=D, dtype=dtype,
                page=page, tree=tree)


def listed():
    """ctx and new are the longest request's; the others are ragged below."""
    return [
        # a decoding step of a full batch: one token a request, long tables
        _tables("tables_step_64", 64, 131071, 1, 16, False),
        # drafts of many requests to verify, each a tree of up to 24 tokens
        _tables("tables_verify_256", 256, 12000, 24, 16, True),
        # prompts of a whole batch given their pages at once
        _tables("tables_prompts_32", 32, 0, 32768, 16, False),
        # a decoding step's keys, values and queries: latency
        _append("append_step_64", 64, 16384, 1, 32, 2, 128, "bfloat16", 16, True),
        # a 32k prompt rotated and written into its pages
        _append("append_prompt_32k", 1, 0, 32768, 32, 2, 128, "bfloat16", 16, True),
        # fp32 rows of head dim 32, an odd number of tokens, larger pages
        _append("append_12k_fp32", 3, 777, 4001, 64, 4, 32, "float32", 64, True),
        # one token of one short request: launches and latency
        _attend("decode_1x2k", 1, 2047, 1, 8, 1, 128, "bfloat16", 16, False),
        # one token each of a ragged batch, groups of 8 heads
        _attend("decode_64x16k", 64, 16383, 1, 32, 4, 128, "bfloat16", 16, False),
        # drafted trees of up to 24 tokens over 32k, groups of 16 heads
        _attend("verify_16x32k", 16, 32768, 24, 32, 2, 128, "bfloat16", 32, True),
        # one long context, a full tree of 64 drafts, 64 heads over 8
        _attend("verify_1x128k", 1, 131008, 64, 64, 8, 128, "bfloat16", 16, True),
        # fp32 with head dim 32 over 120k tokens, five drafts
        _attend("verify_1x120k_fp32", 1, 119995, 5, 64, 4, 32, "float32", 64, True),
        # a chunk of two short ragged fp16 prompts over what is cached
        _attend("chunk_777_fp16", 2, 1500, 777, 8, 2, 64, "float16", 16, False),
    ]


def _log(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))


def draw(rng):
    """A further case of the same ranges: one token to long contexts, trees,
    chains and chunks, every type, groups of 1 to 64 heads."""
    top = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["tables", "append", "attend", "attend"])
        page = rng.choice([16, 16, 32, 64, 128])
        B = _log(rng, 1, 256)
        H, Hkv, D = rng.choice([(32, 2, 128), (32, 4, 128), (64, 8, 128), (64, 4, 32), (8, 1, 128),
                                (8, 2, 64), (16, 4, 32), (4, 1, 64), (64, 1, 64), (6, 2, 96),
                                (16, 2, 256), (4, 4, 128)])
        dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float16", "float32"])
        if op == "tables":
            tree = rng.random() < 0.5
            new = _log(rng, 1, 64 if tree else 16384)
            c = _tables("", B, _log(rng, 1, 131072) - 1, new, page, tree)
        elif op == "append":
            c = _append("", B, _log(rng, 1, 32768) - 1, _log(rng, 1, 16384), H, Hkv, D, dtype, page,
                        rng.random() < 0.8)
        else:
            kind = rng.choice(["decode", "verify", "verify", "chunk"])
            new = 1 if kind == "decode" else _log(rng, 2, 96) if kind == "verify" else _log(rng, 100, 2048)
            c = _attend("", B, _log(rng, 1, 131072) - 1, new, H, Hkv, D, dtype, page, kind == "verify")
            if B * c["ctx"] * Hkv * D > 2 ** 29 or B * H * new * (c["ctx"] + new) > 2 ** 30:
                continue
        if op != "attend" and B * c["new"] > 2 ** 22:
            continue
        if _cost(c) <= top:
            del c["name"]
            return c


def _lengths(c):
    """Per request: tokens in the cache, new ones.  The longest have the
    case's own numbers; without cached tokens some prompts are short too."""
    r = random.Random("%s %s %s %s" % (c["op"], c["B"], c["ctx"], c["new"]))
    ctx = [c["ctx"]] + [r.randint(c["ctx"] // 4, c["ctx"]) for _ in range(c["B"] - 1)]
    new = [c["new"]] + [r.randint(-(-c["new"] // 3), c["new"]) for _ in range(c["B"] - 1)]
    return ctx, new


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


def work(case):
    """Each input read once, each output written once: of the cache the rows
    of the requests, of the tables the entries of those rows."""
    c = case
    ctx, new = _lengths(c)
    rows, page = sum(new), c["page"]
    if c["op"] == "tables":
        had = sum(-(-x // page) for x in ctx)
        now = sum(-(-(x + n) // page) for x, n in zip(ctx, new))
        # lengths in and out, starts, free pages in, entries out, the partly
        # filled pages' entries, slots (8 bytes) and positions of each row
        b = 4 * 4 * c["B"] + 8 * (now - had) + 4 * c["B"] + rows * (12 + 4 * c["tree"])
        return {"bytes": b, "flops": 4 * rows}
    e = 4 if c["dtype"] == "float32" else 2
    H, Hkv, D = c["H"], c["Hkv"], c["D"]
    if c["op"] == "append":
        b = 4 * rows * Hkv * D * e + 8 * rows  # k, v in and out, slots
        if c["rope"]:
            b += 2 * rows * H * D * e + 4 * rows + 4 * D * min(rows, max(x + n for x, n in zip(ctx, new)))
        return {"bytes": b, "flops": 3 * rows * (H + Hkv) * D if c["rope"] else 0}
    keys = sum(x + n for x, n in zip(ctx, new))
    # what a row sees: the cached tokens and, on average, half of a chain or
    # about the depth of a tree
    seen = sum(n * (x + (math.log2(n) + 1 if c["tree"] else (n + 1) / 2)) for x, n in zip(ctx, new))
    b = keys * Hkv * D * 2 * e + 2 * rows * H * D * e + 4 * -(-keys // page) + 4 * rows * c["tree"]
    return {"bytes": b, "flops": int(4 * seen * H * D)}


# ----------------------------------------------------------------- inputs
def _pages(c, seed, spare):
    """Block table of the cached tokens over a shuffled pool, the pool's
    other pages, and how many pages there are."""
    ctx, new = _lengths(c)
    page = c["page"]
    width = max(-(-(x + n) // page) for x, n in zip(ctx, new))
    had = torch.tensor([-(-x // page) for x in ctx])
    now = torch.tensor([-(-(x + n) // page) for x, n in zip(ctx, new)])
    total = int(now.sum()) + spare
    g = torch.Generator(device="cuda").manual_seed(seed)
    pool = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    had = (now if c["op"] != "tables" else had).cuda()
    first = had.cumsum(0) - had
    j = torch.arange(width, device="cuda")
    table = torch.where(j < had[:, None], pool[(first[:, None] + j).clamp(max=total - 1)],
                        torch.full((), -1, dtype=torch.int32, device="cuda")).contiguous()
    return table, pool[int(had.sum()):].contiguous(), total, g


def _tree(c, new, g):
    """A drafted tree for each request: mostly a few branches at each step."""
    n = torch.tensor(new, device="cuda")
    starts = torch.zeros(len(new) + 1, dtype=torch.int32, device="cuda")
    starts[1:] = n.cumsum(0)
    rows = sum(new)
    j = torch.arange(rows, device="cuda") - starts[:-1].long().repeat_interleave(n, output_size=rows)
    back = 1 + (torch.rand(rows, generator=g, device="cuda") ** 2 * torch.clamp(0.5 * j, 4, 12)).long()
    return torch.clamp(j - back, min=-1).to(torch.int32)


def prepare(case, seed):
    c = case
    ctx, new = _lengths(c)
    rows, page = sum(new), c["page"]
    dev = "cuda"
    table, free, pages, g = _pages(c, seed, 7)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    s = dict(op=c["op"], page=page, pages=pages, rows=rows, table=table,
             most=max(x + n for x, n in zip(ctx, new)), most_new=max(new))
    starts = torch.zeros(c["B"] + 1, dtype=torch.int32, device=dev)
    starts[1:] = i32(new).cumsum(0)
    if c["op"] == "tables":
        s.update(ctx=i32(ctx), new=i32(new), free=free,
                 parents=_tree(c, new, g) if c["tree"] else None)
        return s
    t = DTYPES[c["dtype"]]
    H, Hkv, D = c["H"], c["Hkv"], c["D"]
    rand = lambda *n: torch.randn(*n, generator=g, device=dev, dtype=t)
    if c["op"] == "append":
        # packed rows of a fused projection: query, key and value heads
        qkv = rand(rows, H + 2 * Hkv, D)
        s.update(k=qkv[:, H:H + Hkv], v=qkv[:, H + Hkv:], q=None, pos=None, cos=None, sin=None,
                 k_cache=torch.zeros(pages, page, Hkv, D, device=dev, dtype=t),
                 v_cache=torch.zeros(pages, page, Hkv, D, device=dev, dtype=t))
        r = torch.arange(c["B"], device=dev).repeat_interleave(i32(new).long(), output_size=rows)
        at = torch.arange(rows, device=dev) - starts[r].long() + i32(ctx)[r].long()
        s["slots"] = table[r, at // page].long() * page + at % page
        if c["rope"]:
            f = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64, device=dev) / D)
            a = torch.arange(s["most"], dtype=torch.float64, device=dev)[:, None] * f
            s.update(q=qkv[:, :H], pos=at.to(torch.int32), cos=a.cos().float(), sin=a.sin().float())
        return s
    s.update(q=rand(rows, H, D) * 1.5, k_cache=rand(pages, page, Hkv, D),
             v_cache=rand(pages, page, Hkv, D), starts=starts,
             lens=i32([x + n for x, n in zip(ctx, new)]),
             parents=_tree(c, new, g) if c["tree"] else None)
    return s


# ------------------------------------------------------------- plain forms
def _ancestors(parents, starts, n):
    """[B, n, n] 1 where the second index is an ancestor of the first or the
    token itself: the powers of the tree's adjacency, by repeated squaring."""
    B = starts.numel() - 1
    j = torch.arange(n, device=starts.device)
    count = starts.diff()
    row = (starts[:-1, None] + j).clamp(max=parents.numel() - 1)
    p = torch.where(j < count[:, None], parents[row.long()], -1)
    reach = (p[:, :, None] == j).float() + torch.eye(n, device=starts.device)
    for _ in range(max(1, (n - 1).bit_length())):
        reach = torch.matmul(reach, reach).clamp(max=1.0)
    return reach


def _tables_plain(s):
    ctx, new, page, W = s["ctx"].long(), s["new"].long(), s["page"], s["table"].shape[1]
    had, now = (ctx + page - 1) // page, (ctx + new + page - 1) // page
    need = now - had
    first = need.cumsum(0) - need
    j = torch.arange(W, device=ctx.device)
    at = first[:, None] + j - had[:, None]
    fresh = (j >= had[:, None]) & (j < now[:, None])
    s["table"].copy_(torch.where(fresh, s["free"][at.clamp(0, s["free"].numel() - 1)], s["table"]))
    starts = torch.zeros(ctx.numel() + 1, dtype=torch.int64, device=ctx.device)
    starts[1:] = new.cumsum(0)
    row = torch.arange(s["rows"], device=ctx.device)
    r = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    at = ctx[r] + row - starts[r]
    slots = s["table"][r, at // page].long() * page + at % page
    pos = at
    if s["parents"] is not None:
        depth = _ancestors(s["parents"], starts, s["most_new"]).sum(-1).long() - 1
        pos = ctx[r] + depth[r, row - starts[r]]
    return {"table": s["table"], "starts": starts.int(), "slots": slots, "positions": pos.int(),
            "lens": (ctx + new).int(), "pages_used": need.sum().int().reshape(1)}


def _rotate(x, cos, sin):
    a, b = x.float().chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(x.dtype)


def _append_plain(s):
    k, q = s["k"], None
    if s["q"] is not None:
        at = s["pos"].long()
        cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
        k, q = _rotate(k, cos, sin), _rotate(s["q"], cos, sin)
    s["k_cache"].view(-1, *k.shape[1:])[s["slots"]] = k
    s["v_cache"].view(-1, *k.shape[1:])[s["slots"]] = s["v"]
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _attend_plain(s):
    q, kc, vc, table, page = s["q"], s["k_cache"], s["v_cache"], s["table"], s["page"]
    starts, lens, n, L = s["starts"].long(), s["lens"].long(), s["most_new"], s["most"]
    B, (rows, H, D), Hkv = lens.numel(), q.shape, kc.shape[2]
    dev = q.device
    at = torch.arange(L, device=dev)
    there = at < lens[:, None]
    slot = torch.where(there, table[:, at // page].long() * page + at % page, 0)
    keys = kc.view(-1, Hkv, D)[slot].float().permute(0, 2, 3, 1).contiguous()  # [B, Hkv, D, L]
    vals = vc.view(-1, Hkv, D)[slot].float().permute(0, 2, 1, 3).contiguous()
    j = torch.arange(n, device=dev)
    row = (starts[:-1, None] + j).clamp(max=rows - 1)
    qs = q[row].float().view(B, n, Hkv, H // Hkv, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, D)
    ctx = lens - starts.diff()
    i = at - ctx[:, None]  # index among the new tokens
    if s["parents"] is None:
        sees = i[:, None] <= j[:, None]
    else:
        reach = _ancestors(s["parents"], starts, n) > 0
        sees = (i[:, None] < 0) | reach.gather(2, i.clamp(0, n - 1)[:, None].expand(B, n, L))
    sees = (sees & there[:, None])[:, None, :, None]  # [B, 1, n, 1, L]
    x = torch.matmul(qs, keys).view(B, Hkv, n, H // Hkv, L) * D ** -0.5
    x = x.masked_fill(~sees, -math.inf)
    x = x - x.amax(-1, keepdim=True)
    p = x.exp()
    p = (p / p.sum(-1, keepdim=True)).view(B, Hkv, -1, L)
    o = torch.matmul(p, vals).view(B, Hkv, n, H // Hkv, D).permute(0, 2, 1, 3, 4).reshape(B, n, H, D)
    r = torch.searchsorted(starts[1:].contiguous(), torch.arange(rows, device=dev), right=True)
    return o[r, torch.arange(rows, device=dev) - starts[r]].to(q.dtype)


# -------------------------------------------------------------------- run
def run(state):
    s = state
    if own:
        import htree_amd

        if s["op"] == "tables":
            t = htree_amd.page_tables(s["ctx"], s["new"], s["table"], s["free"], s["page"],
                                      s["pages"], s["rows"], parents=s["parents"])
            return {"table": s["table"], "starts": t.starts, "slots": t.slots,
                    "positions": t.positions, "lens": t.lens, "pages_used": t.pages_used}
        if s["op"] == "append":
            q = htree_amd.cache_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"],
                                       q=s["q"], positions=s["pos"], cos=s["cos"], sin=s["sin"])
            return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
        return htree_amd.draft_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"],
                                         s["starts"], parents=s["parents"])
    return {"tables": _tables_plain, "append": _append_plain, "attend": _attend_plain}[s["op"]](s)


# ------------------------------------------------------------------ exact
def exact(case, seed):
    """The definition, request by request, in 64 bits."""
    if case["op"] == "tables":  # whole numbers alone
        return None
    s = prepare(case, seed)
    ctx, new = _lengths(case)
    page = case["page"]
    H, Hkv, D = case["H"], case["Hkv"], case["D"]
    if case["op"] == "append":
        out = {}
        for name in ("k", "v"):
            x = s[name].double()
            if name == "k" and case["rope"]:
                x = _turned(x, s)
            cache = s[name + "_cache"].double().flatten(0, 1)
            cache.index_copy_(0, s["slots"], x)
            out[name + "_cache"] = cache.view(-1, page, Hkv, D)
        return dict(out, q=_turned(s["q"].double(), s) if case["rope"] else None)
    if work(case)["flops"] > 2e13:
        return None
    out = torch.empty(s["rows"], H, D, dtype=torch.float64, device="cuda")
    first = 0
    up = s["parents"].tolist() if case["tree"] else None
    for b in range(case["B"]):
        n, x = new[b], ctx[b]
        pages = s["table"][b, :-(-(x + n) // page)].long()
        k = s["k_cache"][pages].reshape(-1, Hkv, D)[:x + n].double()
        v = s["v_cache"][pages].reshape(-1, Hkv, D)[:x + n].double()
        hide = torch.zeros(n, x + n, dtype=torch.bool)
        hide[:, x:] = True
        for i in range(n):
            if up is None:
                hide[i, x:x + i + 1] = False
                continue
            a = i
            while a >= 0:
                hide[i, x + a] = False
                a = up[first + a]
        hide = hide.cuda()
        for h in range(H):
            w = s["q"][first:first + n, h].double() @ k[:, h * Hkv // H].t() / math.sqrt(D)
            w[hide] = -math.inf
            out[first:first + n, h] = torch.softmax(w, -1) @ v[:, h * Hkv // H]
        first += n
    return out


def _turned(x, s):
    at = s["pos"].long()
    turn = torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None]
    half = x.shape[-1] // 2
    z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * turn
    return torch.cat([z.real, z.imag], -1)

"""GPU tests of page_tables and cache_append against plain implementations:
whole numbers exactly, rotated rows in 64 bits to the bound derived at
`rotation_bar`."""
import numpy as np
import pytest
import torch

import htree_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def i32(x):
    return torch.as_tensor(np.asarray(x, np.int64)).to(torch.int32).to(DEV)


def plain_tables(ctx, new, table, free, page, pages, rows, parents=None):
    """page_tables' definition, request by request (positions and lens end at
    2^31 - 1, the largest an int32 holds)."""
    top = 2 ** 31 - 1
    table = table.copy()
    width = table.shape[1]
    starts, slots, pos, lens, used = [0], np.full(rows, -1, np.int64), np.full(rows, -1, np.int64), [], 0
    for b in range(len(ctx)):
        c = max(int(ctx[b]), 0)
        n = min(max(int(new[b]), 0), rows - starts[-1])
        for j in range(-(-c // page), -(-(c + n) // page)):
            if j < width:
                ok = used < len(free) and 0 <= free[used] < pages
                table[b, j] = free[used] if ok else -1
            used += 1
        for i in range(n):
            r, p = starts[-1] + i, c + i
            if p // page < width and 0 <= table[b, p // page] < pages:
                slots[r] = int(table[b, p // page]) * page + p % page
            depth, a = 0, i
            if parents is None:
                depth = i
            else:
                while 0 <= parents[starts[-1] + a] < a:
                    a = parents[starts[-1] + a]
                    depth += 1
            pos[r] = min(c + depth, top)
        starts.append(starts[-1] + n)
        lens.append(min(c + n, top))
    return table, np.array(starts), slots, pos, np.array(lens), used


def check_tables(ctx, new, width, page, pages, rows, free, parents=None, table=None, stride=None):
    g = np.random.default_rng(5)
    B = len(ctx)
    if table is None:
        table = g.integers(0, max(pages, 1), (B, width))
        for b in range(B):
            table[b, -(-max(int(ctx[b]), 0) // page):] = -1
    want = plain_tables(ctx, new, table, free, page, pages, rows, parents)
    dev = torch.full((B, stride or width), -7, dtype=torch.int32, device=DEV)
    view = dev[:, :width]
    view.copy_(i32(table))
    for _ in range(2):  # in place: the same again
        t = htree_amd.page_tables(i32(ctx), i32(new), view, i32(free), page, pages, rows,
                                  parents=None if parents is None else i32(parents))
        torch.cuda.synchronize()
        got = (view, t.starts, t.slots, t.positions, t.lens, t.pages_used)
        for name, a, b in zip(("table", "starts", "slots", "positions", "lens", "pages_used"), got, want):
            assert np.array_equal(a.cpu().numpy().astype(np.int64).reshape(-1), np.asarray(b).reshape(-1)), name
    if stride:
        assert bool((dev[:, width:] == -7).all())
    return t


@pytest.mark.parametrize("B,ctx_most,new_most,page", [
    (1, 0, 1, 16), (1, 100, 1, 16), (3, 40, 40, 16), (64, 500, 1, 16), (65, 300, 33, 32), (257, 200, 9, 16),
    (700, 50, 5, 1), (5, 0, 3001, 128), (4096, 40, 2, 16), (2, 70000, 20000, 64)])
def test_tables_match_definition(B, ctx_most, new_most, page):
    g = np.random.default_rng(B + page)
    ctx, new = g.integers(0, ctx_most + 1, B), g.integers(0, new_most + 1, B)
    new[0], ctx[-1] = new_most, ctx_most
    rows = int(new.sum()) + 3
    width = max(-(-int(c + n) // page) for c, n in zip(ctx, new)) + 1
    pages = int((-(-(ctx + new) // page)).sum()) + 4
    free = g.permutation(pages)
    check_tables(ctx, new, width, page, pages, rows, free, stride=width + 5)


@pytest.mark.parametrize("shape", ["random", "chain", "star", "damaged"])
@pytest.mark.parametrize("new", [[1], [0, 24, 7], [64] * 20, [3, 1500, 2]])
def test_tables_of_drafted_trees(shape, new):
    g = np.random.default_rng(len(new))
    rows = sum(new)
    idx = np.concatenate([np.arange(n) for n in new]).astype(np.int64)
    parents = {"random": np.array([g.integers(-1, j) if j else -1 for j in idx]), "chain": idx - 1,
               "star": np.full(rows, -1), "damaged": g.integers(-5, 80, rows)}[shape]
    ctx = g.integers(0, 100, len(new))
    check_tables(ctx, new, 120, 16, 400, rows, g.permutation(400), parents)


def test_tables_damaged_inputs():
    """Negative and huge lengths, pages out of range in the table and the
    list, too few pages, a narrow table, too few rows."""
    g = np.random.default_rng(1)
    ctx, new = np.array([5, -3, 40, 2 ** 31 - 1, 17, 16]), np.array([20, 4, -2, 3, 2, 100])
    table = g.integers(-3, 30, (6, 4))
    free = np.array([3, 25, -1, 7, 2 ** 31 - 1, 8])
    check_tables(ctx, new, 4, 16, 20, 160, free, table=table)
    check_tables(ctx, new, 4, 16, 20, 25, free, table=table)    # rows run out
    check_tables(ctx, new, 4, 16, 20, 160, free[:0], table=table)
    check_tables(ctx, new, 0, 16, 20, 160, free, table=table[:, :0])


def test_tables_out_and_empty():
    t = check_tables([5], [3], 2, 16, 9, 4, [2, 1])
    again = htree_amd.page_tables(i32([15]), i32([3]), i32([[4, -1]]), i32([2, 1]), 16, 9, 4, out=t)
    torch.cuda.synchronize()
    assert again.slots is t.slots
    assert t.slots.tolist() == [79, 32, 33, -1] and t.pages_used.tolist() == [1]
    e = htree_amd.page_tables(i32([]), i32([]), i32(np.zeros((0, 3))), i32([1]), 16, 9, 2)
    assert e.starts.tolist() == [0] and e.slots.tolist() == [-1, -1] and e.lens.numel() == 0
    z = check_tables([5, 20], [0, 0], 2, 16, 9, 0, [2, 1])
    assert z.slots.numel() == 0


# ---------------------------------------------------------------- append
def rotation_bar(x, cos, sin, dtype):
    """|error| of a rotated element: two products and a sum in fp32 (2^-24 of
    each term, twice), then one rounding of at most half a step."""
    h = x.shape[-1] // 2
    a, b = np.abs(x[..., :h]), np.abs(x[..., h:])
    c, s = np.abs(cos), np.abs(sin)
    size = np.concatenate([a * c + b * s, b * c + a * s], -1)
    half = torch.finfo(DT[dtype]).eps / 2
    tiny = torch.finfo(DT[dtype]).tiny * torch.finfo(DT[dtype]).eps  # half a step of subnormals, at most
    return size * (half * (1 + 2.0 ** -22) + 2.0 ** -22) + tiny


def rotated(x, cos, sin):
    h = x.shape[-1] // 2
    return np.concatenate([x[..., :h] * cos - x[..., h:] * sin, x[..., h:] * cos + x[..., :h] * sin], -1)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("rows,H,Hkv,K,V", [(1, 8, 1, 128, 128), (7, 32, 2, 128, 64), (130, 6, 2, 96, 96),
                                            (33, 64, 4, 32, 32), (5, 5, 5, 256, 256), (300, 4, 1, 24, 40),
                                            (2000, 16, 4, 64, 64), (11, 100, 3, 8, 16)])
@pytest.mark.parametrize("rope", [True, False])
def test_append(dtype, rows, H, Hkv, K, V, rope):
    t = DT[dtype]
    g = torch.Generator().manual_seed(rows + K)
    page, pages = 16, rows // 16 + 9
    qkv = torch.randn(rows, H + 2 * Hkv, max(K, V), generator=g).to(t).to(DEV)
    q, k, v = qkv[:, :H, :K], qkv[:, H:H + Hkv, :K], qkv[:, H + Hkv:, :V]
    kc = torch.full((pages, page, Hkv, K), 7.0, dtype=t, device=DEV)
    vc = torch.full((pages, Hkv, page, V), 7.0, dtype=t, device=DEV).permute(0, 2, 1, 3)  # heads before tokens
    slots = torch.randperm(pages * page, generator=g)[:rows]
    dead = torch.rand(rows, generator=g) < 0.1
    slots[dead] = torch.tensor([-1, pages * page, 2 ** 40, -2 ** 40])[torch.arange(rows) % 4][dead]
    pos = torch.randint(0, 500, (rows,), generator=g)
    lost = torch.rand(rows, generator=g) < 0.1
    if rope:
        pos[lost] = torch.tensor([-1, 500, 2 ** 31 - 1])[torch.arange(rows) % 3][lost]
    cos, sin = htree_amd.rope_cache(K, 500, 10000.0, DEV)
    kw = dict(q=q, positions=pos.int().to(DEV), cos=cos, sin=sin) if rope else {}
    qo = htree_amd.cache_append(k, v, kc, vc, slots.to(DEV), **kw)
    torch.cuda.synchronize()
    n = lambda x: x.double().cpu().numpy()
    at = pos.clamp(0, 499).numpy()
    c, s = n(cos)[at][:, None], n(sin)[at][:, None]
    writes = ~dead & ~(lost if rope else torch.zeros_like(lost))
    want_k = np.full((pages * page, Hkv, K), 7.0)
    want_v = np.full((pages * page, Hkv, V), 7.0)
    bar = np.zeros_like(want_k)
    sl = slots[writes].numpy()
    w = writes.numpy()
    want_k[sl] = rotated(n(k), c, s)[w] if rope else n(k)[w]
    want_v[sl] = n(v)[w]
    if rope:
        bar[sl] = rotation_bar(n(k), c, s, dtype)[w]
    got_k, got_v = n(kc.reshape(-1, Hkv, K)), n(vc.reshape(-1, Hkv, V))
    assert np.array_equal(got_v, want_v)
    assert np.all(np.abs(got_k - want_k) <= bar)
    if rope:
        want_q = np.where(lost.numpy()[:, None, None], 0.0, rotated(n(q), c, s))
        assert qo.shape == (rows, H, K) and qo.is_contiguous()
        assert np.all(np.abs(n(qo) - want_q) <= rotation_bar(n(q), c, s, dtype))
    else:
        assert qo is None


def test_append_odd_strides_are_copied():
    """Rows the kernels cannot read in 16-byte pieces: transposed, misaligned,
    expanded over heads."""
    base = torch.randn(32 * 9 * 2 + 8, device=DEV)
    k = base[1:1 + 9 * 64].view(9, 2, 32)                  # 4 bytes off
    v = torch.randn(9, 32, 2, device=DEV).transpose(1, 2)  # head dim strided
    for kk, vv in ((k, v), (torch.randn(9, 1, 32, device=DEV).expand(9, 2, 32), k)):
        kc, vc = torch.zeros(2, 16, 2, 32, device=DEV), torch.zeros(2, 16, 2, 32, device=DEV)
        slots = torch.randperm(32)[:9].to(DEV)
        htree_amd.cache_append(kk, vv, kc, vc, slots)
        assert torch.equal(kc.view(-1, 2, 32)[slots], kk) and torch.equal(vc.view(-1, 2, 32)[slots], vv)
        assert int((kc.view(-1, 64).abs().sum(1) > 0).sum()) == 9


def test_append_past_32_bits():
    """A cache of more than 2^32 bytes, written at both ends."""
    pages = 70000
    kc = torch.empty(pages, 16, 16, 128, dtype=torch.bfloat16, device=DEV)
    vc = torch.empty(pages, 16, 16, 128, dtype=torch.bfloat16, device=DEV)
    assert kc.numel() * 2 > 2 ** 32
    k, v = torch.randn(2, 4, 16, 128, device=DEV).bfloat16()
    slots = torch.tensor([0, pages * 16 - 1, pages * 8 + 3, 65535 * 16 + 9], device=DEV)
    htree_amd.cache_append(k, v, kc, vc, slots)
    assert torch.equal(kc.view(-1, 16, 128)[slots], k) and torch.equal(vc.view(-1, 16, 128)[slots], v)


def test_refusals():
    f = lambda *n, t=torch.bfloat16: torch.zeros(n, dtype=t, device=DEV)
    kc, sl = f(4, 16, 2, 64), torch.zeros(3, dtype=torch.int64, device=DEV)
    k = f(3, 2, 64)
    pos, cs = i32([0, 1, 2]), torch.zeros(8, 32, device=DEV)
    ap = htree_amd.cache_append
    bad = [
        lambda: ap(k, k, kc, f(4, 16, 1, 64), sl), lambda: ap(k.float(), k, kc, kc, sl),
        lambda: ap(f(3, 1, 64), k, kc, kc, sl), lambda: ap(k, k, kc, kc, sl.int()),
        lambda: ap(k, k, kc, kc, sl[:2]), lambda: ap(k, k, f(4, 8, 2, 64), f(4, 8, 2, 64), sl),
        lambda: ap(k, k, kc[:1].expand(4, 16, 2, 64), kc, sl), lambda: ap(k, k, kc, kc, sl, q=k),
        lambda: ap(k, k, kc, kc, sl, positions=pos), lambda: ap(k, k, kc, kc, sl, positions=pos, cos=cs),
        lambda: ap(k, k, kc, kc, sl, positions=pos, cos=cs[:, :8], sin=cs[:, :8]),
        lambda: ap(k, k, kc, kc, sl, positions=sl, cos=cs, sin=cs),
        lambda: ap(k.clone().requires_grad_(), k, kc, kc, sl),
        lambda: ap(f(3, 2, 60), f(3, 2, 60), f(4, 16, 2, 60), f(4, 16, 2, 60), sl),
        lambda: htree_amd.page_tables(sl, i32([1, 1, 1]), i32(np.zeros((3, 2))), i32([1]), 16, 2, 3),
        lambda: htree_amd.page_tables(i32([1]), i32([1, 1]), i32(np.zeros((1, 2))), i32([1]), 16, 2, 3),
        lambda: htree_amd.page_tables(i32([1]), i32([1]), i32(np.zeros((2, 2))), i32([1]), 16, 2, 3),
        lambda: htree_amd.page_tables(i32([1]), i32([1]), i32(np.zeros((1, 2))), i32([1]), 12, 2, 3),
        lambda: htree_amd.page_tables(i32([1]), i32([1]), i32(np.zeros((1, 2))), i32([1]), 16, 2, -1),
        lambda: htree_amd.page_tables(i32([1]), i32([1]), i32(np.zeros((1, 2))), i32([1]), 16, 2, 3, parents=i32([1])),
    ]
    t = htree_amd.page_tables(i32([1]), i32([1]), i32(np.zeros((1, 2))), i32([1]), 16, 2, 3)
    bad += [  # the last step's lengths as input of the next, written in place
        lambda: htree_amd.page_tables(t.lens, i32([1]), i32(np.zeros((1, 2))), i32([1]), 16, 2, 3, out=t),
        lambda: htree_amd.page_tables(i32([1]), i32([1]), i32(np.zeros((1, 2))), i32([1]), 16, 2, 3,
                                      parents=t.positions, out=t),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(AssertionError):
            call()
            print("not refused:", i)

"""cache_append from rows that lie in the cache itself: the C entry refuses
them (a row could be read after another one's write), Python copies them
before anything is written."""
import ctypes

import pytest
import torch

import htree_amd
from htree_amd import _native as N

BASE = 1 << 20  # never read: the calls are refused


def call(rows=4, k=BASE, v=BASE, q=None, kc=BASE, vc=BASE, k_row=256, q_row=512):
    """H_kv 2, D 128, bf16: rows of 512 bytes; caches of 8 pages of 16 tokens,
    64 KB each; q has 4 heads, 1024 bytes a row."""
    c = N.HtreeCache(1, 2, 128, 128, 16, 8, 16 * 256, 256, 128, 16 * 256, 256, 128)
    p = lambda x: ctypes.c_void_p(x)
    tab = p(BASE) if q else None
    return N.lib().htree_cache_append(c, rows, 4 if q else 0, p(k), k_row, 128, p(v), 256, 128, p(q), q_row, 128,
                                      p(BASE), tab, tab, tab, 8 if q else 0, tab, p(kc), p(vc), None)


FAR, SIZE = 1 << 30, 8 * 16 * 512


@pytest.mark.parametrize("what", ["k", "v", "q"])
@pytest.mark.parametrize("cache", ["kc", "vc"])
@pytest.mark.parametrize("shift", [0, 16, SIZE - 16, -16, -4 * 512 + 16])
def test_the_c_entry_refuses_rows_of_the_cache(what, cache, shift):
    at = {"k": 2 * FAR, "v": 3 * FAR, "q": 4 * FAR, "kc": 5 * FAR, "vc": 6 * FAR}
    at[what] = at[cache] + shift
    assert call(**at) == N.HTREE_EOVERLAP
    assert "cache" in N.strerror(N.HTREE_EOVERLAP)


def test_strided_rows_count_with_their_gaps():
    assert call(k=BASE, v=3 * FAR, kc=BASE + 4096, vc=6 * FAR, rows=4, k_row=4096) == N.HTREE_EOVERLAP


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,shift", [(1000, 3), (1000, -3), (5000, 1), (40, 700)])
@pytest.mark.parametrize("rope", [False, True])
def test_rows_moved_within_the_cache(dtype, rows, shift, rope):
    """Keys and values moved by a few slots, as views; with a rotation, the
    queries from the value cache."""
    pages, Hkv, D = -(-rows // 16) + 60, 2, 64
    dev = "cuda:0"
    g = torch.Generator().manual_seed(rows)
    kc, vc = (torch.randn(pages, 16, Hkv, D, generator=g).to(dtype).to(dev) for _ in range(2))
    kf, vf = kc.view(-1, Hkv, D), vc.view(-1, Hkv, D)
    at = 10
    slots = torch.arange(at + shift, at + shift + rows, device=dev)
    cos, sin = htree_amd.rope_cache(D, 99, 10000.0, dev)
    pos = torch.randint(0, 99, (rows,), generator=g, dtype=torch.int32).to(dev)

    def go(copy):
        k2, v2 = kc.clone(), vc.clone()
        k, v = k2.view(-1, Hkv, D)[at:at + rows], v2.view(-1, Hkv, D)[at:at + rows]
        q = v2.view(-1, Hkv, D)[:rows]
        if copy:
            k, v, q = k.clone(), v.clone(), q.clone()
        r = htree_amd.cache_append(k, v, k2, v2, slots, **(dict(q=q, positions=pos, cos=cos, sin=sin) if rope else {}))
        return (k2, v2, r) if rope else (k2, v2)

    want = go(True)
    if not rope:
        wk, wv = kf.clone(), vf.clone()
        wk[slots], wv[slots] = kf[at:at + rows], vf[at:at + rows]
        assert torch.equal(want[0].view(-1, Hkv, D), wk) and torch.equal(want[1].view(-1, Hkv, D), wv)
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(go(False), want))


@pytest.mark.gpu
def test_neighbours_are_no_overlap():
    """Rows right before and right behind the caches, and caches of one
    buffer, keys beside values in a page: the same as apart."""
    dev, n, D = "cuda:0", 32, 64
    buf = torch.randn(4 * n, 1, D, device=dev)
    k, kc, v = buf[:n], buf[n:3 * n].view(4, 16, 1, D), buf[3 * n:]
    vc = torch.zeros(4, 16, 1, D, device=dev)
    slots = torch.randperm(2 * n, device=dev)[:n]
    k0, v0 = k.clone(), v.clone()
    htree_amd.cache_append(k, v, kc, vc, slots)
    assert torch.equal(kc.view(-1, 1, D)[slots], k0) and torch.equal(vc.view(-1, 1, D)[slots], v0)
    assert torch.equal(k, k0) and torch.equal(v, v0)
    both = torch.zeros(4, 2, 16, 1, D, device=dev)
    htree_amd.cache_append(k, v, both[:, 0], both[:, 1], slots)
    assert torch.equal(both[:, 0].reshape(-1, 1, D)[slots], k0) and torch.equal(both[:, 1].reshape(-1, 1, D)[slots], v0)


@pytest.mark.parametrize("name", ["ctx", "new", "parents", "free"])
@pytest.mark.parametrize("over", ["table", "starts", "slots", "positions", "lens", "used"])
def test_page_tables_refuses_inputs_that_it_writes(name, over):
    """4 requests, 6 rows, 3 pages, a table of 4 x 10."""
    at = {n: (i + 1) * FAR for i, n in enumerate(("ctx", "new", "parents", "free", "table", "starts", "slots",
                                                 "positions", "lens", "used"))}
    size = dict(table=160, starts=20, slots=48, positions=24, lens=16, used=4)[over]
    for shift in (0, size - 4):
        at[name] = at[over] + shift
        p = lambda n: ctypes.c_void_p(at[n])
        assert N.lib().htree_page_tables(4, 6, 16, 9, 10, 10, 3, p("ctx"), p("new"), p("parents"), p("table"),
                                         p("free"), p("starts"), p("slots"), p("positions"), p("lens"), p("used"),
                                         None) == N.HTREE_EOVERLAP


@pytest.mark.parametrize("over", ["starts", "slots", "positions", "lens", "used"])
def test_page_tables_refuses_outputs_in_the_table(over):
    at = {n: (i + 1) * FAR for i, n in enumerate(("ctx", "new", "parents", "free", "table", "starts", "slots",
                                                 "positions", "lens", "used"))}
    at[over] = at["table"] + 156
    p = lambda n: ctypes.c_void_p(at[n])
    assert N.lib().htree_page_tables(4, 6, 16, 9, 10, 10, 3, p("ctx"), p("new"), p("parents"), p("table"), p("free"),
                                     p("starts"), p("slots"), p("positions"), p("lens"), p("used"),
                                     None) == N.HTREE_EOVERLAP


@pytest.mark.gpu
def test_a_captured_move():
    """The copies are part of the capture: every replay moves the rows as they
    are then."""
    dev, n, D = "cuda:0", 100, 64
    g = torch.Generator().manual_seed(5)
    kc, vc = torch.zeros(12, 16, 2, D, device=dev), torch.zeros(12, 16, 2, D, device=dev)
    kf, vf = kc.view(-1, 2, D), vc.view(-1, 2, D)
    slots = torch.arange(3, 3 + n, device=dev)
    call = lambda k, v: htree_amd.cache_append(kf[:n], vf[:n], k, v, slots)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(kc, vc)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(kc, vc)
    for _ in range(4):
        kc.copy_(torch.randn(kc.shape, generator=g))
        vc.copy_(torch.randn(vc.shape, generator=g))
        wk, wv = kf.clone(), vf.clone()
        wk[slots], wv[slots] = kf[:n].clone(), vf[:n].clone()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kf, wk) and torch.equal(vf, wv)

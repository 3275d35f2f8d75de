"""Serving from a paged key/value cache: block tables and slot maps from
request lengths, and new keys and values (rotated by their positions) written
to their slots.  The attention over the cache is draft.py's.

The reference has no serving path (its entry points take whole sequences,
/root/reference/src/parallel.py:874-885); this one carries on where its
forward ends: up to max_top_nodes tokens a sequence's tree has one level and
htree_forward is dense causal attention with RoPE at the token's position
(src/parallel.py:941-945, 983-988), whose next rows come from the cache.

The cache is two tensors that the caller keeps, k_cache
[pages, page_size, H_kv, K] and v_cache [pages, page_size, H_kv, V] (any
strides that are whole 16-byte pieces, the head dim contiguous: a permuted
[pages, H_kv, page_size, K] tensor serves too).  Token p of request b is in
page block_table[b, p // page_size] at offset p % page_size; a slot is
page * page_size + offset.

Lengths, tables, slots and positions stay on the GPU and are not checked by
the host; whatever they hold, the kernels touch nothing outside the tensors.
Nothing here synchronises, so a step can be captured into a graph.
"""
from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _native as N

MAX_REQUESTS = 4096
MAX_HEAD_DIM = 256
PAGE_SIZES = (16, 4096)       # of the cache: powers of two in this range
MAX_REQUEST_TOKENS = 1 << 30  # block table width * page_size
MAX_TOKEN_BYTES = 1 << 26     # between a page's tokens
INT32 = 1 << 31               # sizes below: the C ABI's are int32


class PageTables(NamedTuple):
    """What page_tables returns, int32 but for the slots (int64)."""
    starts: torch.Tensor      # [B + 1] first row of each request
    slots: torch.Tensor       # [rows] slot of each new token, -1: none
    positions: torch.Tensor   # [rows] its position (depth in a drafted tree)
    lens: torch.Tensor        # [B] tokens in the cache, the new ones included
    pages_used: torch.Tensor  # [1] pages taken from the front of free_pages


def _ints(t: torch.Tensor, name: str, n: int, device) -> None:
    assert t.dtype is torch.int32 and t.shape == (n,) and t.is_contiguous(), \
        f"{name} must be a contiguous int32 tensor [{n}], got {t.dtype} {list(t.shape)}"
    assert t.device == device, f"{name} must be on {device}"


def overlap(a: torch.Tensor, b: Optional[torch.Tensor]) -> bool:
    """Whether two tensors' memory, gaps included, overlaps."""
    def end(t):
        return t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()
    return b is not None and a.numel() > 0 and b.numel() > 0 and a.data_ptr() < end(b) and b.data_ptr() < end(a)


def no_derivatives(name: str, *tensors: Optional[torch.Tensor]) -> None:
    """Refuses tensors whose gradient or forward-mode tangent a call would lose."""
    if torch.is_grad_enabled():
        for t in tensors:
            assert t is None or not t.requires_grad, f"{name} has no backward"
    no_tangents(name, *tensors)


def no_tangents(name: str, *tensors: Optional[torch.Tensor]) -> None:
    """Refuses tensors whose forward-mode tangent a call would lose."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            assert t is None or forward_ad.unpack_dual(t).tangent is None, f"{name} has no forward-mode derivative"


def check_table(block_table: torch.Tensor, B: int, device) -> None:
    assert block_table.dtype is torch.int32 and block_table.dim() == 2, "block_table must be int32 [B, width]"
    assert block_table.shape[0] == B, f"block_table must have a row for each of the {B} requests"
    assert block_table.stride(1) == 1 or block_table.shape[1] <= 1 or B == 0, "block_table rows must be contiguous"
    assert B <= 1 or block_table.stride(0) >= block_table.shape[1], "block_table must not be expanded"
    assert block_table.device == device, f"block_table must be on {device}"


def aligned_rows(x: torch.Tensor) -> torch.Tensor:
    """x [rows, heads, D] itself where the kernels can read it: the head dim
    contiguous, rows and heads at 16-byte steps; else a contiguous copy."""
    n, h, d = x.stride()
    if (d == 1 or x.shape[2] == 1) and ((n | h) * x.element_size() | x.data_ptr()) % 16 == 0:
        return x
    return x.clone(memory_format=torch.contiguous_format)


@lru_cache(maxsize=256)
def _describe(kshape, kstride, vshape, vstride, dtype) -> "N.HtreeCache":
    """The cache's sizes for the C ABI, checked (by sizes and strides alone)."""
    assert len(kshape) == 4 and len(vshape) == 4, "k_cache / v_cache must be [pages, page_size, H_kv, D]"
    pages, page, heads, K = kshape
    V = vshape[3]
    assert vshape[:3] == kshape[:3], "k_cache and v_cache must have the same pages and heads"
    assert dtype in N.DTYPE_CODE, "the cache's dtype must be float32, bfloat16 or float16"
    assert 0 < pages < INT32 and 0 < heads < INT32, "the cache needs a page and a head, and less than 2^31 of either"
    assert PAGE_SIZES[0] <= page <= PAGE_SIZES[1] and page & (page - 1) == 0, \
        f"page_size must be a power of two from {PAGE_SIZES[0]} to {PAGE_SIZES[1]}, got {page}"
    es = dtype.itemsize
    assert 0 < K <= MAX_HEAD_DIM and 0 < V <= MAX_HEAD_DIM and K * es % 16 == 0 and V * es % 16 == 0, \
        f"head dims must be whole 16-byte pieces and at most {MAX_HEAD_DIM}, got K={K}, V={V}"
    assert kstride[3] == 1 and vstride[3] == 1, "the cache's head dim must be contiguous"
    assert all(n * es % 16 == 0 for n in kstride[:3] + vstride[:3]), \
        "the cache's pages, tokens and heads must be at 16-byte steps"
    assert kstride[1] * es <= MAX_TOKEN_BYTES and vstride[1] * es <= MAX_TOKEN_BYTES, \
        f"a page's tokens must be at most {MAX_TOKEN_BYTES} bytes apart"
    return N.HtreeCache(N.DTYPE_CODE[dtype], heads, K, V, page, pages, *kstride[:3], *vstride[:3])


def native_cache(k_cache: torch.Tensor, v_cache: torch.Tensor) -> "N.HtreeCache":
    """Checks the cache tensors and describes them for the C ABI."""
    dtype, dev = k_cache.dtype, k_cache.device
    assert dev.type == "cuda", "htree_amd runs on the GPU (no CPU fallback)"
    assert v_cache.dtype is dtype, "k_cache and v_cache must share one dtype"
    assert v_cache.device == dev, "k_cache and v_cache must be on one device"
    assert (k_cache.data_ptr() | v_cache.data_ptr()) % 16 == 0, "the cache must begin at a 16-byte step"
    return _describe(k_cache.shape, k_cache.stride(), v_cache.shape, v_cache.stride(), dtype)


def page_tables(ctx_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor,
                free_pages: torch.Tensor, page_size: int, num_pages: int, rows: int,
                parents: Optional[torch.Tensor] = None, out: Optional[PageTables] = None) -> PageTables:
    """Room for a step's new tokens, worked out on the GPU.

    Request b has ctx_lens[b] tokens in the cache and gets new_lens[b] more
    (int32 [B]).  The pages it lacks are taken from the front of free_pages
    (int32 [F]), request after request, and entered in block_table
    (int32 [B, width], in place: its other entries stay).  `rows` is the
    number of new tokens there is room for, at least the sum of new_lens in
    the common case; tokens past it are dropped.  parents (int32 [rows])
    makes the new tokens of a request drafted trees: parents[row] is the
    index, within the request, of the token drafted before it, a smaller one
    (-1: none); positions are then those along each branch.

    Returns PageTables (`out`: written there; it does not overlap the
    inputs).  Rows behind the last request
    have slot and position -1; so has the slot of a token past the table's
    width, or whose page free_pages was too short for (pages_used says how
    many are wanted).  page_size is a power of two."""
    dev = ctx_lens.device
    assert dev.type == "cuda", "htree_amd runs on the GPU (no CPU fallback)"
    assert ctx_lens.dim() == 1 and free_pages.dim() == 1, "ctx_lens and free_pages must be int32 [B] and [F]"
    B, F = ctx_lens.shape[0], free_pages.shape[0]
    assert B <= MAX_REQUESTS, f"at most {MAX_REQUESTS} requests, got {B}"
    _ints(ctx_lens, "ctx_lens", B, dev)
    _ints(new_lens, "new_lens", B, dev)
    _ints(free_pages, "free_pages", F, dev)
    check_table(block_table, B, dev)
    assert page_size > 0 and page_size & (page_size - 1) == 0, f"page_size must be a power of two, got {page_size}"
    assert 0 <= rows < INT32 and 0 <= num_pages < INT32, "rows and num_pages must not be negative, nor pass 31 bits"
    assert page_size < INT32 and F < INT32 and block_table.shape[1] < INT32, \
        "page_size, free_pages and block_table's width must not pass 31 bits"
    if parents is not None:
        _ints(parents, "parents", rows, dev)
    if out is None:
        starts, positions, lens, used = torch.empty(2 * B + 2 + rows, dtype=torch.int32, device=dev).split_with_sizes(
            (B + 1, rows, B, 1))
        out = PageTables(starts, torch.empty(rows, dtype=torch.int64, device=dev), positions, lens, used)
    else:
        _ints(out.starts, "out.starts", B + 1, dev)
        _ints(out.positions, "out.positions", rows, dev)
        _ints(out.lens, "out.lens", B, dev)
        _ints(out.pages_used, "out.pages_used", 1, dev)
        assert out.slots.dtype is torch.int64 and out.slots.shape == (rows,) and out.slots.is_contiguous() \
            and out.slots.device == dev, f"out.slots must be a contiguous int64 tensor [{rows}] on {dev}"
    if B == 0:
        out.starts.zero_(), out.pages_used.zero_(), out.slots.fill_(-1), out.positions.fill_(-1)
        return out
    rc = N.launch(N.lib().htree_page_tables, dev, B, rows, page_size, num_pages, block_table.shape[1],
                  block_table.stride(0), F, ctx_lens.data_ptr(), new_lens.data_ptr(), N.address(parents),
                  block_table.data_ptr(), free_pages.data_ptr(), out.starts.data_ptr(), out.slots.data_ptr(),
                  out.positions.data_ptr(), out.lens.data_ptr(), out.pages_used.data_ptr())
    if rc:
        assert rc != N.HTREE_EOVERLAP, "out and block_table, which are written, must not overlap the inputs"
        N.check(rc, "htree_page_tables")
    return out


def cache_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 slots: torch.Tensor, q: Optional[torch.Tensor] = None,
                 positions: Optional[torch.Tensor] = None, cos: Optional[torch.Tensor] = None,
                 sin: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Writes new tokens' keys k [rows, H_kv, K] and values v [rows, H_kv, V]
    into the cache at slots (int64 [rows], as page_tables gives them).

    With the tables cos / sin (fp32 [n, K/2], htree_amd.rope_cache) each key
    is rotated by its row's position (int32 [rows]) first, pairs
    (d, d + K/2) as in htree_forward, and the queries q [rows, H, K] with
    them: the rotated queries are returned (None without q).  Products and
    sums are fp32, rounded once.  Rows whose slot or position is out of range
    are not written, and a query without a position is zero.  The slots of a
    call are distinct; two rows with one slot leave either's values there,
    or parts of both.  k, v and q may be parts of the cache: where their
    memory's range overlaps its, they are copied before anything is written."""
    c = native_cache(k_cache, v_cache)
    dtype, dev = k_cache.dtype, k_cache.device
    assert k.dim() == 3 and v.dim() == 3, "k / v must be [rows, H_kv, D]"
    rows = k.shape[0]
    assert rows < INT32, f"rows must be below 2^31, got {rows}"
    assert k.shape == (rows, c.H_kv, c.Dk) and v.shape == (rows, c.H_kv, c.Dv), \
        f"k / v must be [rows, {c.H_kv}, {c.Dk} / {c.Dv}], got {list(k.shape)} / {list(v.shape)}"
    assert k.dtype is dtype and v.dtype is dtype, "k, v and the cache must share one dtype"
    assert k.device == dev and v.device == dev, "k, v and the cache must be on one device"
    for n, x, y in zip(k_cache.shape, k_cache.stride(), v_cache.stride()):
        assert n == 1 or (x > 0 and y > 0), "k_cache and v_cache must not be expanded"
    assert slots.dtype is torch.int64 and slots.shape == (rows,) and slots.is_contiguous() \
        and slots.device == dev, f"slots must be a contiguous int64 tensor [{rows}] on {dev}"
    no_derivatives("cache_append", k, v, q, cos, sin, k_cache, v_cache)
    assert (cos is None) == (sin is None) == (positions is None), "positions, cos and sin go together"
    H, rope_rows, q_out, q_row, q_head = 0, 0, None, 0, 0
    if cos is not None:
        assert c.Dk % 2 == 0, "rotating needs an even head dim K"
        rope_rows, half = cos.shape[0], c.Dk // 2
        assert 0 < rope_rows < INT32 and cos.shape == (rope_rows, half) and sin.shape == (rope_rows, half) \
            and cos.dtype is torch.float32 and sin.dtype is torch.float32 \
            and cos.is_contiguous() and sin.is_contiguous() and cos.device == dev and sin.device == dev, \
            f"cos and sin must be contiguous fp32 tensors [n, {half}] on {dev}"
        _ints(positions, "positions", rows, dev)
    if q is not None:
        assert cos is not None, "q is taken to be rotated: it needs positions, cos and sin"
        assert q.dim() == 3 and q.shape[0] == rows and q.shape[2] == c.Dk and 0 < q.shape[1] < INT32, \
            f"q must be [{rows}, H, {c.Dk}], got {list(q.shape)}"
        assert q.dtype is dtype and q.device == dev, "q must have k's dtype and device"
        H = q.shape[1]
        q = aligned_rows(q)
        q_out = torch.empty((rows, H, c.Dk), dtype=dtype, device=dev)
    k, v = aligned_rows(k), aligned_rows(v)
    for copied in (False, True):
        if copied:
            k, v, q = (None if x is None else x.clone(memory_format=torch.contiguous_format) for x in (k, v, q))
        k_row, k_head, _ = k.stride()
        v_row, v_head, _ = v.stride()
        if q is not None:
            q_row, q_head, _ = q.stride()
        rc = N.launch(N.lib().htree_cache_append, dev, c, rows, H, k.data_ptr(), k_row, k_head, v.data_ptr(), v_row,
                      v_head, N.address(q), q_row, q_head, slots.data_ptr(), N.address(positions), N.address(cos),
                      N.address(sin), rope_rows, N.address(q_out), k_cache.data_ptr(), v_cache.data_ptr())
        if rc != N.HTREE_EOVERLAP:
            break
    if rc:
        N.check(rc, "htree_cache_append")
    return q_out

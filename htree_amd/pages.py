"""Pages of the serving cache after a step: accepted drafts moved together,
requests forked (samples of one prompt, beams), pages copied, and the pages
that no request holds, for the next step's page_tables.

Caches are given for one layer, k_caches [pages, page_size, H_kv, K] as
cache.py has it, or for all layers at once: one tensor [layers, pages, ...]
or a sequence of a tensor each, alike in sizes and strides.  They may lie in one
buffer, in any order, but no two entries in the same place.  All layers move in
one launch.  Nothing here synchronises."""
from __future__ import annotations

import ctypes
from array import array
from functools import lru_cache
from typing import NamedTuple, Optional, Sequence, Union

import torch

from . import _native as N
from .cache import INT32, MAX_REQUESTS, _describe, _ints, check_table, no_derivatives

Caches = Union[torch.Tensor, Sequence[torch.Tensor]]
MAX_LAYERS = 65535
MAX_COPIES = 1 << 24
_SHARED = "each layer's keys and values must have memory of their own, apart from the lists, and not be expanded"


class Forked(NamedTuple):
    """What fork_requests returns, int32."""
    block_table: torch.Tensor  # [N, width]
    lens: torch.Tensor         # [N] tokens of each new request
    copy_from: torch.Tensor    # [N] page whose tokens it needs a copy of, -1: none
    copy_to: torch.Tensor      # [N] its own page for them
    copy_tokens: torch.Tensor  # [N] how many
    pages_used: torch.Tensor   # [1] pages taken from the front of free_pages


class UnusedPages(NamedTuple):
    """What unused_pages returns, int32."""
    pages: torch.Tensor  # [num_pages] ascending, -1 behind the last one
    count: torch.Tensor  # [1]


def _bases(caches: Caches, name: str):
    """A layer's shape and stride, a tensor of its type and device, and the
    address of each layer."""
    if isinstance(caches, torch.Tensor):
        shape, stride, at = caches.shape, caches.stride(), caches.data_ptr()
        if len(shape) == 4:
            return shape, stride, caches, (at,)
        assert len(shape) == 5, f"{name} must be [pages, page_size, H_kv, D] or [layers, pages, page_size, H_kv, D]"
        layers, step = shape[0], stride[0] * caches.element_size()
        assert 0 < layers <= MAX_LAYERS, f"{name} must have 1 to {MAX_LAYERS} layers"
        assert layers == 1 or step > 0, f"{name} must not be expanded"
        return shape[1:], stride[1:], caches, range(at, at + layers * step, step) if step else (at,)
    caches = list(caches)
    assert 0 < len(caches) <= MAX_LAYERS, f"{name} must have 1 to {MAX_LAYERS} layers"
    first = caches[0]
    shape, stride, dtype, dev = first.shape, first.stride(), first.dtype, first.device
    for c in caches:
        assert c.dim() == 4 and c.shape == shape and c.stride() == stride and c.dtype is dtype and c.device == dev, \
            f"the layers of {name} must be alike: sizes, strides, type and device"
    return shape, stride, first, [c.data_ptr() for c in caches]


@lru_cache(maxsize=256)
def _layout(kshape, kstride, vshape, vstride, dtype) -> "N.HtreeCache":
    """The description of layers that are written to."""
    c = _describe(kshape, kstride, vshape, vstride, dtype)
    for size, a, b in zip(kshape, kstride, vstride):
        assert size == 1 or (a > 0 and b > 0), "k_caches and v_caches must not be expanded"
    return c


def _layers(name: str, k_caches: Caches, v_caches: Caches):
    """Checks the layers; their description and addresses for the C ABI."""
    ks, kt, k, k_at = _bases(k_caches, "k_caches")
    vs, vt, v, v_at = _bases(v_caches, "v_caches")
    dev, n = k.device, len(k_at)
    assert dev.type == "cuda", "htree_amd runs on the GPU (no CPU fallback)"
    assert v.dtype is k.dtype and v.device == dev, "k_caches and v_caches must share one dtype and device"
    assert len(v_at) == n, f"k_caches and v_caches must have as many layers, got {n} and {len(v_at)}"
    c = _layout(ks, kt, vs, vt, k.dtype)
    assert len({*k_at, *v_at}) == 2 * n, "each layer's keys and values must be tensors of their own"
    if k is k_caches and v is v_caches:
        no_derivatives(name, k, v)
    else:
        for x in (k_caches, v_caches):
            no_derivatives(name, *((x,) if isinstance(x, torch.Tensor) else x))
    k_ptr, v_ptr = array("Q", k_at), array("Q", v_at)
    return c, n, k_ptr, v_ptr, dev


def keep_drafts(k_caches: Caches, v_caches: Caches, slots: torch.Tensor, starts: torch.Tensor,
                path: torch.Tensor, kept: torch.Tensor) -> None:
    """Moves the accepted drafts of a step to the front of their request's new
    tokens in the cache, so that the request's next lengths are the cached
    tokens it had and kept[b].

    slots (int64 [rows]) and starts (int32 [B + 1]) are the step's
    (page_tables), path (int32 [rows]) and kept (int32 [B]) verify_drafts':
    what is in slot slots[starts[b] + path[starts[b] + j]] goes to slot
    slots[starts[b] + j], for every j below kept[b].  path ascends within a
    request, so path[j] >= j; entries that are smaller than j, or not of the
    request, are left out, and so are slots outside the cache.  The slots of a
    step are distinct, its pages no other request's."""
    c, layers, k_ptr, v_ptr, dev = _layers("keep_drafts", k_caches, v_caches)
    assert slots.dim() == 1 and kept.dim() == 1, "slots must be int64 [rows] and kept int32 [B]"
    rows, B = slots.shape[0], kept.shape[0]
    assert rows < INT32, f"rows must be below 2^31, got {rows}"
    assert B <= MAX_REQUESTS, f"at most {MAX_REQUESTS} requests, got {B}"
    assert slots.dtype is torch.int64 and slots.is_contiguous() and slots.device == dev, \
        f"slots must be a contiguous int64 tensor [rows] on {dev}"
    _ints(starts, "starts", B + 1, dev)
    _ints(path, "path", rows, dev)
    _ints(kept, "kept", B, dev)
    rc = N.launch(N.lib().htree_keep_drafts, dev, c, layers, k_ptr.buffer_info()[0], v_ptr.buffer_info()[0], B, rows, slots.data_ptr(),
                  starts.data_ptr(), path.data_ptr(), kept.data_ptr())
    if rc:
        assert rc != N.HTREE_EOVERLAP, _SHARED
        N.check(rc, "htree_keep_drafts")


def copy_pages(k_caches: Caches, v_caches: Caches, copy_from: torch.Tensor, copy_to: torch.Tensor,
               copy_tokens: Optional[torch.Tensor] = None) -> None:
    """Copies page copy_from[i] to page copy_to[i] (int32 [n]), its first
    copy_tokens[i] tokens (int32 [n]; without them whole pages), in every
    layer: what fork_requests asks for, or pages moved to others.  Pages
    outside the cache (-1) are left out.  No page is in copy_to twice, nor in
    both lists."""
    c, layers, k_ptr, v_ptr, dev = _layers("copy_pages", k_caches, v_caches)
    assert copy_from.dim() == 1, "copy_from must be int32 [n]"
    n = copy_from.shape[0]
    assert n < MAX_COPIES, f"pages to copy must be less than {MAX_COPIES}, got {n}"
    _ints(copy_from, "copy_from", n, dev)
    _ints(copy_to, "copy_to", n, dev)
    if copy_tokens is not None:
        _ints(copy_tokens, "copy_tokens", n, dev)
    rc = N.launch(N.lib().htree_copy_pages, dev, c, layers, k_ptr.buffer_info()[0], v_ptr.buffer_info()[0], n,
                  copy_from.data_ptr(), copy_to.data_ptr(), N.address(copy_tokens))
    if rc:
        assert rc != N.HTREE_EOVERLAP, _SHARED
        N.check(rc, "htree_copy_pages")


def _sizes(page_size: int, num_pages: int, block_table: torch.Tensor) -> None:
    assert 0 < page_size < INT32 and page_size & (page_size - 1) == 0, \
        f"page_size must be a power of two below 2^31, got {page_size}"
    assert 0 <= num_pages < INT32 and block_table.shape[1] < INT32, \
        "num_pages and block_table's width must not pass 31 bits"


def fork_requests(block_table: torch.Tensor, lens: torch.Tensor, source: torch.Tensor,
                  free_pages: torch.Tensor, page_size: int, num_pages: int,
                  out: Optional[Forked] = None) -> Forked:
    """New requests that carry on from others: samples of one prompt, beams
    that go on, in any order and number.

    New request i has the tokens of request source[i] (int32 [N]; a number
    outside 0 .. B - 1 makes an empty one), lens[source[i]] of them (int32
    [B]), in the pages of block_table (int32 [B, width]).  Full pages are
    shared.  A partly filled last page stays with the first new request of
    its source; each further one gets a fresh page from the front of
    free_pages (int32 [F], as page_tables takes them), into which copy_pages
    copies the page's tokens, before either request is appended to.  Requests
    that share pages are not cut back into them: their lengths do not go below
    what they were forked at.

    Returns Forked (`out`: written there; no overlap with the inputs).
    Entries behind a request's last page are -1, and so is a page that
    free_pages was too short for (pages_used says how many are wanted).  The
    requests that source leaves out are gone: their pages are in
    unused_pages' list after this."""
    dev = lens.device
    assert dev.type == "cuda", "htree_amd runs on the GPU (no CPU fallback)"
    assert lens.dim() == 1 and source.dim() == 1 and free_pages.dim() == 1, \
        "lens, source and free_pages must be int32 [B], [N] and [F]"
    B, n, F = lens.shape[0], source.shape[0], free_pages.shape[0]
    assert B <= MAX_REQUESTS and n <= MAX_REQUESTS, f"at most {MAX_REQUESTS} requests, got {B} and {n}"
    assert F < INT32, "free_pages must not pass 31 bits"
    _ints(lens, "lens", B, dev)
    _ints(source, "source", n, dev)
    _ints(free_pages, "free_pages", F, dev)
    check_table(block_table, B, dev)
    _sizes(page_size, num_pages, block_table)
    width = block_table.shape[1]
    if out is None:
        out = Forked(block_table.new_empty((n, width)),
                     *source.new_empty(4 * n + 1).split_with_sizes((n, n, n, n, 1)))
    else:
        check_table(out.block_table, n, dev)
        assert out.block_table.shape[1] == width, f"out.block_table must be [{n}, {width}]"
        for name, t in zip(Forked._fields[1:], out[1:]):
            _ints(t, f"out.{name}", 1 if name == "pages_used" else n, dev)
    if n == 0:
        out.pages_used.zero_()
        return out
    rc = N.launch(N.lib().htree_fork_requests, dev, B, n, page_size, num_pages, width, block_table.stride(0),
                  out.block_table.stride(0), F, block_table.data_ptr(), lens.data_ptr(), source.data_ptr(),
                  free_pages.data_ptr(), out.block_table.data_ptr(), out.lens.data_ptr(), out.copy_from.data_ptr(),
                  out.copy_to.data_ptr(), out.copy_tokens.data_ptr(), out.pages_used.data_ptr())
    if rc:
        assert rc != N.HTREE_EOVERLAP, "out must not overlap the inputs, nor its parts each other"
        N.check(rc, "htree_fork_requests")
    return out


@lru_cache(maxsize=64)
def _unused_workspace_bytes(B: int, num_pages: int, width: int, held: int) -> int:
    n = ctypes.c_int64()
    N.check(N.lib().htree_unused_pages_workspace_bytes(B, num_pages, width, held, n), "htree_unused_pages_workspace_bytes")
    return n.value


def unused_pages(block_table: torch.Tensor, lens: torch.Tensor, page_size: int, num_pages: int,
                 held: Optional[torch.Tensor] = None, out: Optional[UnusedPages] = None) -> UnusedPages:
    """The pages of a pool of num_pages that no request holds: those in none
    of the entries 0 .. ceil(lens[b] / page_size) - 1 of block_table (int32
    [B, width]) and not among held (int32 [M]; pages of requests that wait, or
    kept for later prompts; -1: none).  A request is freed by a length of 0,
    what a step did not keep by a shorter one; pages that forked requests
    share are held until the last of them is gone.

    Returns UnusedPages (`out`: written there; no overlap with the inputs).
    The list is in ascending order and as long as the pool, -1 behind the
    last page: page_tables and fork_requests take it as it is."""
    dev = lens.device
    assert dev.type == "cuda", "htree_amd runs on the GPU (no CPU fallback)"
    assert lens.dim() == 1, "lens must be int32 [B]"
    B = lens.shape[0]
    assert B <= MAX_REQUESTS, f"at most {MAX_REQUESTS} requests, got {B}"
    _ints(lens, "lens", B, dev)
    check_table(block_table, B, dev)
    _sizes(page_size, num_pages, block_table)
    M = 0
    if held is not None:
        assert held.dim() == 1 and held.shape[0] < INT32, "held must be int32 [M]"
        M = held.shape[0]
        _ints(held, "held", M, dev)
    if out is None:
        out = UnusedPages(*lens.new_empty(num_pages + 1).split_with_sizes((num_pages, 1)))
    else:
        _ints(out.pages, "out.pages", num_pages, dev)
        _ints(out.count, "out.count", 1, dev)
    if num_pages == 0:
        out.count.zero_()
        return out
    width = block_table.shape[1]
    nbytes = _unused_workspace_bytes(B, num_pages, width, M)
    ws = lens.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    rc = N.launch(N.lib().htree_unused_pages, dev, B, page_size, num_pages, width, block_table.stride(0), block_table.data_ptr(), lens.data_ptr(), M, N.address(held),
                  out.pages.data_ptr(), out.count.data_ptr(), N.address(ws), nbytes)
    if rc:
        assert rc != N.HTREE_EOVERLAP, "out must not overlap the inputs, nor its parts each other"
        N.check(rc, "htree_unused_pages")
    return out

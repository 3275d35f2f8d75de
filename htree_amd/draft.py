"""Attention of new tokens over a paged key/value cache: one token of each
request (decoding), drafted trees of tokens to verify, or chunks of prompts.
The cache, block tables and slots are cache.py's."""
from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional

import torch

from . import _native as N
from .cache import (INT32, MAX_REQUEST_TOKENS, MAX_REQUESTS, _ints, aligned_rows, check_table, native_cache,
                    no_derivatives, overlap)

MAX_SCALE = 2.35e38  # scale * log2(e) is an fp32 number


@lru_cache(maxsize=256)
def _workspace_bytes(sizes, B: int, rows: int, H: int, width: int) -> int:
    n = ctypes.c_int64()
    N.check(N.lib().htree_draft_attention_workspace_bytes(N.HtreeCache(*sizes), B, rows, H, width, n),
            "htree_draft_attention_workspace_bytes")
    return n.value


def draft_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    block_table: torch.Tensor, lens: torch.Tensor, starts: torch.Tensor,
                    parents: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale q k^T) v over what each row sees of its request.

    q [rows, H, K]: the new tokens of all requests, rows starts[b] ..
    starts[b + 1] - 1 (int32 [B + 1]) those of request b.  Their keys and
    values are in the cache already (cache_append), the last of the lens[b]
    tokens (int32 [B]) of the request.  Row j of a request sees the tokens
    before the new ones, its ancestors by parents (int32 [rows]: the index
    within the request of the token drafted before it, a smaller one, -1:
    none) and itself; without parents the new tokens up to itself.  (Branches
    are walked token by token: drafts of tens or hundreds of tokens.  A chunk
    of thousands belongs in a call without parents: a chain of 2048 takes
    9 ms instead of 0.3, and at least four times that for twice the tokens.)
    scale defaults to K^-0.5, and is at most MAX_SCALE in size.  Queries and
    keys come rotated.

    Returns [rows, H, V] in q's dtype (`out`: written there, contiguous, no
    overlap with the inputs).  Rows that see nothing are zero, and so are
    those all of whose scores are -inf; rows behind the last request are not
    written.  Pages outside the cache hold no tokens, neither does the request
    past its table.

    Scores and the softmax are fp32 (fp32 products for fp32 inputs); for
    16-bit types P is rounded to the type for the product with the values
    (fp16: each weight to half a step, or 2^-36 of the row's largest).
    At most MAX_REQUESTS requests: each block sums all of their lengths.
    Results do not depend on the other requests' values, but a request's
    split, and so the last bits, depends on all lengths."""
    c = native_cache(k_cache, v_cache)
    dtype, dev = k_cache.dtype, k_cache.device
    assert q.dim() == 3, "q must be [rows, H, K]"
    rows, H, K = q.shape
    assert K == c.Dk, f"q and the cache must share the head dim K ({K} vs {c.Dk})"
    assert rows < INT32 and H < INT32, f"rows and heads must be below 2^31, got {rows} and {H}"
    assert H > 0 and H % c.H_kv == 0, f"H ({H}) must be divisible by H_kv ({c.H_kv})"
    assert q.dtype is dtype, "q and the cache must share one dtype"
    assert q.device == dev, "q and the cache must be on one device"
    assert lens.dim() == 1, "lens must be int32 [B]"
    B = lens.shape[0]
    assert B <= MAX_REQUESTS, f"at most {MAX_REQUESTS} requests, got {B}"
    _ints(lens, "lens", B, dev)
    _ints(starts, "starts", B + 1, dev)
    check_table(block_table, B, dev)
    width = block_table.shape[1]
    assert width * c.page_size <= MAX_REQUEST_TOKENS, \
        f"a request's table holds at most {MAX_REQUEST_TOKENS} tokens, got {width * c.page_size}"
    if parents is not None:
        _ints(parents, "parents", rows, dev)
    no_derivatives("draft_attention", q, k_cache, v_cache, out)
    if out is None:
        out = torch.empty((rows, H, c.Dv), dtype=dtype, device=dev)
    else:
        assert out.shape == (rows, H, c.Dv) and out.dtype is dtype and out.is_contiguous() \
            and out.device == dev and out.data_ptr() % 16 == 0, \
            f"out must be a contiguous {dtype} tensor [{rows}, {H}, {c.Dv}] on {dev}"
        assert not any(overlap(out, x) for x in (q, k_cache, v_cache, block_table, lens, starts, parents)), \
            "out must not overlap the inputs"
    scale = K ** -0.5 if scale is None else float(scale)
    assert abs(scale) <= MAX_SCALE, f"scale must be a number of at most {MAX_SCALE} in size, got {scale}"
    if B == 0 or rows == 0:
        return out
    q = aligned_rows(q)
    q_row, q_head, _ = q.stride()
    nbytes = _workspace_bytes((c.dtype, c.H_kv, K, c.Dv, c.page_size, c.num_pages, c.k_page, c.k_token, c.k_head,
                               c.v_page, c.v_token, c.v_head), B, rows, H, width)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    rc = N.launch(N.lib().htree_draft_attention, dev, c, B, rows, H, width, block_table.stride(0),
                  scale, q.data_ptr(), q_row, q_head, k_cache.data_ptr(),
                  v_cache.data_ptr(), block_table.data_ptr(), lens.data_ptr(), starts.data_ptr(), N.address(parents),
                  out.data_ptr(), H * c.Dv, c.Dv, N.address(ws), nbytes)
    if rc:
        N.check(rc, "htree_draft_attention")
    return out

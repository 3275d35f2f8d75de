"""Verification of drafted tokens: which of them the target's probabilities
accept, from given uniform numbers, and the token after the last one.  The
drafts are those that draft.py's attention was computed for; pages.py moves
the kept ones together."""
from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import NamedTuple, Optional

import torch

from . import _native as N
from .cache import INT32, MAX_REQUESTS, _ints

MAX_DRAFT_ROWS = 1024  # of a request that are looked at


class Verified(NamedTuple):
    """What verify_drafts returns."""
    kept: torch.Tensor         # [B] int32: rows kept, the first one of the request included
    path: torch.Tensor         # [rows] int32: from starts[b] on their indices within the request, -1 elsewhere
    next_tokens: torch.Tensor  # [B] int64: the token after the last kept row


@lru_cache(maxsize=256)
def _workspace_bytes(dtype, B: int, rows: int, V: int, drawn: bool, greedy: bool) -> int:
    n = ctypes.c_int64()
    N.check(N.lib().htree_verify_drafts_workspace_bytes(N.DTYPE_CODE[dtype], B, rows, V, drawn, greedy, n),
            "htree_verify_drafts_workspace_bytes")
    return n.value


def _probs(p: torch.Tensor, name: str, rows: int, V: int, dtype, device) -> None:
    assert p.shape == (rows, V) and p.dtype is dtype and p.device == device, \
        f"{name} must be a {dtype} tensor [{rows}, {V}] on {device}, got {p.dtype} {list(p.shape)}"
    assert p.stride(1) == 1 or V == 1, f"{name}'s rows must be contiguous"


def verify_drafts(target_probs: torch.Tensor, tokens: torch.Tensor, starts: torch.Tensor,
                  uniforms: Optional[torch.Tensor] = None, draws: Optional[torch.Tensor] = None,
                  draft_probs: Optional[torch.Tensor] = None, parents: Optional[torch.Tensor] = None,
                  out: Optional[Verified] = None) -> Verified:
    """Accepts or rejects drafted tokens so that what is kept is distributed
    as the target's own tokens would be.

    Rows starts[b] .. starts[b + 1] - 1 (int32 [B + 1]) are request b's new
    tokens (tokens, int64 [rows]), as page_tables and draft_attention take
    them.  The first is the token its last step decided on, and is kept.  The
    others are drafts: row j was drafted after row parents[j] of its request
    (int32 [rows]: a smaller index), without parents after the row before.  A
    row without such a parent, or whose token is not in the vocabulary, is
    not kept, nor is anything drafted after it.

    target_probs [rows, V] are the target's probabilities after each row
    (float32, bfloat16 or float16; a row sums to one).  A kept row's drafts
    are tried in order, with T the target's probabilities there and S = 1:
      with draft_probs [rows, V], the drafter's probabilities after each row,
        from which its drafts were drawn independently, with replacement (one
        token may come twice): draft c of token x is accepted if
        uniforms[c] S q(x) < T(x); a rejected one leaves T = max(T - S q, 0)
        and S = sum T to the next;
      without them (drafts chosen in any way, the likeliest for instance or
        siblings drawn without replacement, for which draft_probs would give
        another distribution): accepted if uniforms[c] S < T(x); a rejected one
        leaves T(x) = 0, and S less what T(x) was.
    An accepted draft is kept and its own drafts follow.  Where none is
    accepted, or there are none, the next token is drawn from T: the first
    whose cumulative T passes draws[b] sum T (if nothing is left of T, from
    the target's probabilities).  uniforms (float32 [rows]; those of first
    rows are not used) and draws (float32 [B]) are from [0, 1).

    Without uniforms, draws and draft_probs the drafts are verified greedily:
    one is accepted if its token is that of the largest entry after the row
    it was drafted after, and that token is the next one where none is.
    target_probs may be any scores then; of equal entries the first counts, a
    NaN does not.

    Sums are 64-bit.  Entries that are no positive finite numbers count as
    zero, and so do uniforms and draws that are not positive.  A request
    without rows keeps 0 and has next token -1; without any mass (greedily: any
    entry above -infinity) the next token is -1 too.  Of a request the first
    MAX_DRAFT_ROWS rows are looked at.

    Returns Verified (`out`: written there; no overlap with the inputs).
    Nothing synchronises; the numbers are the same every run."""
    dev = target_probs.device
    assert dev.type == "cuda", "htree_amd runs on the GPU (no CPU fallback)"
    assert target_probs.dim() == 2, "target_probs must be [rows, V]"
    rows, V = target_probs.shape
    dtype = target_probs.dtype
    assert dtype in N.DTYPE_CODE, "target_probs must be float32, bfloat16 or float16"
    assert rows < INT32 and 0 < V < INT32, f"rows and the vocabulary must be below 2^31, got {rows} and {V}"
    _probs(target_probs, "target_probs", rows, V, dtype, dev)
    if draft_probs is not None:
        _probs(draft_probs, "draft_probs", rows, V, dtype, dev)
    assert starts.dim() == 1 and starts.shape[0] > 0, "starts must be int32 [B + 1]"
    B = starts.shape[0] - 1
    assert B <= MAX_REQUESTS, f"at most {MAX_REQUESTS} requests, got {B}"
    _ints(starts, "starts", B + 1, dev)
    greedy = uniforms is None
    assert greedy == (draws is None), "uniforms and draws go together"
    if greedy:
        assert draft_probs is None, "draft_probs need uniforms and draws"
    else:
        for t, name, n in ((uniforms, "uniforms", rows), (draws, "draws", B)):
            assert t.dtype is torch.float32 and t.shape == (n,) and t.is_contiguous() and t.device == dev, \
                f"{name} must be a contiguous float32 tensor [{n}] on {dev}"
    assert tokens.dtype is torch.int64 and tokens.shape == (rows,) and tokens.is_contiguous() and tokens.device == dev, \
        f"tokens must be a contiguous int64 tensor [{rows}] on {dev}"
    if parents is not None:
        _ints(parents, "parents", rows, dev)
    if out is None:
        like = draws if draws is not None else starts[1:]
        out = Verified(torch.empty_like(like, dtype=torch.int32), torch.empty_like(tokens, dtype=torch.int32),
                       torch.empty_like(like, dtype=torch.int64))
    else:
        _ints(out.kept, "out.kept", B, dev)
        _ints(out.path, "out.path", rows, dev)
        assert out.next_tokens.dtype is torch.int64 and out.next_tokens.shape == (B,) \
            and out.next_tokens.is_contiguous() and out.next_tokens.device == dev, \
            f"out.next_tokens must be a contiguous int64 tensor [{B}] on {dev}"
    if B == 0:
        out.path.fill_(-1)
        return out
    nbytes = _workspace_bytes(dtype, B, rows, V, draft_probs is not None, greedy)
    ws = starts.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    rc = N.launch(N.lib().htree_verify_drafts, dev, N.DTYPE_CODE[dtype], B, rows, V, target_probs.data_ptr(),
                  target_probs.stride(0), N.address(draft_probs), 0 if draft_probs is None else draft_probs.stride(0),
                  tokens.data_ptr(), starts.data_ptr(), N.address(parents), N.address(uniforms), N.address(draws),
                  out.kept.data_ptr(), out.path.data_ptr(), out.next_tokens.data_ptr(), N.address(ws), nbytes)
    if rc:
        assert rc != N.HTREE_EOVERLAP, "out must not overlap the inputs, nor its parts each other"
        N.check(rc, "htree_verify_drafts")
    return out

"""htree_amd: hierarchical tree sparse attention on MI355X (gfx950).

Drop-in for the reference's src/parallel.py / src/backward.py entry points:
    htree_forward(q, k, v, compression_rate, max_top_nodes, top_k_per_layer,
                  scale, rope_base, _save_for_backward, _save_parents, _save_scores)
    htree_backward(dO, q, output, bwd_ctx) -> (dq, dk, dv)
    htree_forward_triton_autograd(q, k, v, ...)   (name kept for drop-in use;
                                                   runs the HIP kernels)
and the trace harness of correctness_test.py:
    run_parallel_with_trace(...) -> (output, trace), LayerTrace, compare_traces
and, for serving, attention of new tokens over a paged key/value cache:
    page_tables(ctx_lens, new_lens, block_table, free_pages, ...) -> PageTables
    cache_append(k, v, k_cache, v_cache, slots, q, positions, cos, sin) -> rotated q
    draft_attention(q, k_cache, v_cache, block_table, lens, starts, parents)
with what surrounds it in a step:
    head_norm(q, k, q_weight, k_weight, ...) -> (q, k)   (for training too)
    verify_drafts(target_probs, tokens, starts, uniforms, draws, ...) -> Verified
    keep_drafts(k_caches, v_caches, slots, starts, path, kept)
    fork_requests(block_table, lens, source, free_pages, ...) -> Forked
    copy_pages(k_caches, v_caches, copy_from, copy_to, copy_tokens)
    unused_pages(block_table, lens, page_size, num_pages, held) -> UnusedPages
"""
from .parallel import (HTREE_SCORE_NEG_INF, HTREE_SCORE_VALID_THRESHOLD, htree_forward,
                       htree_forward_parents, rope_cache)
from .backward import (HTreeFunction, HTreeLeanFunction, HTreeScoresFunction, HTreeTritonFunction,
                       htree_backward, htree_forward_autograd, htree_forward_triton_autograd)
from .trace import LayerTrace, compare_traces, run_parallel_with_trace
from .topk import topk_rows
from .cache import PageTables, cache_append, page_tables
from .draft import draft_attention
from .norm import head_norm
from .pages import Forked, UnusedPages, copy_pages, fork_requests, keep_drafts, unused_pages
from .verify import Verified, verify_drafts


__all__ = [
    "htree_forward", "htree_forward_parents", "htree_backward", "htree_forward_triton_autograd",
    "htree_forward_autograd", "HTreeTritonFunction", "HTreeScoresFunction", "HTreeLeanFunction",
    "HTreeFunction", "rope_cache",
    "HTREE_SCORE_NEG_INF", "HTREE_SCORE_VALID_THRESHOLD", "LayerTrace", "run_parallel_with_trace",
    "compare_traces", "topk_rows", "PageTables", "page_tables", "cache_append", "draft_attention",
    "head_norm", "Verified", "verify_drafts", "keep_drafts", "Forked", "fork_requests", "copy_pages",
    "UnusedPages", "unused_pages",
]

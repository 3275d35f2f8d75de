"""Norms of queries and keys by head, rotated by their positions in the same
pass: before htree_forward in training (which rotates by itself), before
cache_append in serving."""
from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _native as N
from .cache import INT32, MAX_HEAD_DIM, aligned_rows, no_tangents


@lru_cache(maxsize=16)
def _workspace_bytes(D: int) -> int:
    n = ctypes.c_int64()
    N.check(N.lib().htree_head_norm_backward_workspace_bytes(D, n), "htree_head_norm_backward_workspace_bytes")
    return n.value


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x as the kernels read it: [rows, heads, D], rows and heads at 16-byte steps."""
    return aligned_rows(x if x.dim() == 3 else x.reshape(-1, *x.shape[-2:]))


def _codes(q: torch.Tensor, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor]):
    """The inputs' type and the weights'."""
    w = k_weight if q_weight is None else q_weight
    code = N.DTYPE_CODE[q.dtype]
    return code, code if w is None else N.DTYPE_CODE[w.dtype]


def _forward(q, k, q_weight, k_weight, eps, positions, cos, sin):
    """The outputs, and q and k as the kernels read them."""
    dev = q.device
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    q3, k3 = _rows(q), _rows(k)
    rows, H, D = q3.shape
    if rows:
        (qr, qh, _), (kr, kh, _) = q3.stride(), k3.stride()
        rc = N.launch(N.lib().htree_head_norm, dev, *_codes(q, q_weight, k_weight), rows, H, k3.shape[1], D, eps,
                      q3.data_ptr(), qr, qh, k3.data_ptr(), kr, kh, N.address(q_weight), N.address(k_weight),
                      N.address(positions), N.address(cos), N.address(sin), 0 if cos is None else cos.shape[0],
                      q_out.data_ptr(), k_out.data_ptr())
        if rc:
            N.check(rc, "htree_head_norm")
    return q_out, k_out, q3, k3


class _HeadNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, eps, positions, cos, sin):
        ctx.set_materialize_grads(False)
        q_out, k_out, q3, k3 = _forward(q, k, q_weight, k_weight, eps, positions, cos, sin)
        ctx.save_for_backward(q3, k3, q_weight, k_weight, positions, cos, sin)
        ctx.eps, ctx.shapes, ctx.codes = eps, (q.shape, k.shape), _codes(q, q_weight, k_weight)
        return q_out, k_out

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight, positions, cos, sin = ctx.saved_tensors
        needs, dev, (rows, H, D), H_kv = ctx.needs_input_grad, q.device, q.shape, k.shape[1]
        dq = dk = dq_weight = dk_weight = ws = None
        new = torch.empty_like if rows else torch.zeros_like
        qr = qh = kr = kh = yr = yh = zr = zh = nbytes = 0
        if dq_out is None or not (needs[0] or needs[2]):
            q, dq_out, H = None, None, 0
        else:
            dq_out = _rows(dq_out)
            dq = q.new_empty(ctx.shapes[0])
            dq_weight = new(q_weight) if needs[2] else None
            (qr, qh, _), (yr, yh, _) = q.stride(), dq_out.stride()
        if dk_out is None or not (needs[1] or needs[3]):
            k, dk_out, H_kv = None, None, 0
        else:
            dk_out = _rows(dk_out)
            dk = k.new_empty(ctx.shapes[1])
            dk_weight = new(k_weight) if needs[3] else None
            (kr, kh, _), (zr, zh, _) = k.stride(), dk_out.stride()
        if rows and (H or H_kv):
            if dq_weight is not None or dk_weight is not None:
                nbytes = _workspace_bytes(D)
                ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            ptr = N.address
            rc = N.launch(N.lib().htree_head_norm_backward, dev, *ctx.codes, rows, H, H_kv, D, ctx.eps, ptr(q), qr, qh,
                          ptr(k), kr, kh, ptr(dq_out), yr, yh, ptr(dk_out), zr, zh, ptr(q_weight), ptr(k_weight),
                          ptr(positions), ptr(cos), ptr(sin), 0 if cos is None else cos.shape[0], ptr(dq), ptr(dk),
                          ptr(dq_weight), ptr(dk_weight), ptr(ws), nbytes)
            if rc:
                N.check(rc, "htree_head_norm_backward")
        return (dq if needs[0] else None, dk if needs[1] else None, dq_weight, dk_weight, None, None, None, None)


def _check_weight(name: str, w: torch.Tensor, D: int, dtype, dev) -> None:
    assert w.shape == (D,) and (w.dtype is torch.float32 or w.dtype is dtype) and w.is_contiguous() \
        and w.device == dev, f"{name} must be a contiguous [{D}] tensor, float32 or {dtype}, on {dev}"


def head_norm(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
              k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
              positions: Optional[torch.Tensor] = None, cos: Optional[torch.Tensor] = None,
              sin: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Each head's x (mean x^2 + eps)^-1/2 weight, of queries q [..., H, D] and
    keys k [..., H_kv, D] ([rows, H, D] in serving, [B, T, H, D] in training).

    q_weight and k_weight ([D], both float32 or both of q's dtype; None: ones)
    are shared by the heads.  With positions (int32 [...], one a row) and the
    tables cos / sin (fp32 [n, D/2], htree_amd.rope_cache) heads are rotated
    as cache_append rotates them, pairs (d, d + D/2); cache_append and
    draft_attention then take the results as they are.  htree_forward rotates
    by itself: there positions stay out.  Rows whose position is outside the
    tables are zero.

    Products and sums are fp32, rounded once at the end; sizes of up to 1e18
    (their squares are summed).  D is at most 256, in whole 16-byte pieces;
    inputs at other steps than 16 bytes are copied first, and so are those
    whose leading dims are no one step apart.  Rows times heads are below 2^31,
    and times the lanes that a head takes below 2^32: the least power of two of
    at least D / 8 (fp32; D / 16 else), or D / 4 (D / 8) where half a head is no
    whole 16-byte pieces.  Returns contiguous tensors.

    Gradients of q, k and the weights: dx = r (g - x r^2 mean(g x)) with g the
    output's gradient rotated back, times the weight; the weights' are summed
    over rows and heads in fp32, in a fixed order.  There is no second
    derivative and no forward mode; cos and sin have no gradient."""
    dev, dtype, shape, kshape = q.device, q.dtype, q.shape, k.shape
    assert dev.type == "cuda", "htree_amd runs on the GPU (no CPU fallback)"
    assert dtype in N.DTYPE_CODE, "q must be float32, bfloat16 or float16"
    assert k.dtype is dtype and k.device == dev, "q and k must share one dtype and device"
    lead = shape[:-2]
    assert len(shape) >= 3 and len(shape) == len(kshape) and lead == kshape[:-2] and shape[-1] == kshape[-1], \
        f"q and k must be [..., H, D] and [..., H_kv, D], got {list(shape)} and {list(kshape)}"
    H, D, H_kv = shape[-2], shape[-1], kshape[-2]
    assert 0 < D <= MAX_HEAD_DIM and D * dtype.itemsize % 16 == 0, \
        f"the head dim must be whole 16-byte pieces and at most {MAX_HEAD_DIM}, got {D}"
    assert H > 0 and H_kv > 0, "q and k need a head each"
    assert lead.numel() * (H + H_kv) < INT32, "rows times heads must be below 2^31"
    assert 0.0 <= eps < 3.4e38, f"eps must not be negative, nor infinite, got {eps}"
    if q_weight is not None:
        _check_weight("q_weight", q_weight, D, dtype, dev)
    if k_weight is not None:
        _check_weight("k_weight", k_weight, D, dtype, dev)
        assert q_weight is None or q_weight.dtype is k_weight.dtype, "q_weight and k_weight must share one dtype"
    assert (cos is None) == (sin is None) == (positions is None), "positions, cos and sin go together"
    if cos is not None:
        n, half = cos.shape[0], D // 2
        assert 0 < n < INT32 and cos.shape == (n, half) and sin.shape == (n, half) \
            and cos.dtype is torch.float32 and sin.dtype is torch.float32 and cos.is_contiguous() \
            and sin.is_contiguous() and cos.device == dev and sin.device == dev, \
            f"cos and sin must be contiguous fp32 tensors [n, {half}] on {dev}"
        assert positions.dtype is torch.int32 and positions.shape == lead and positions.is_contiguous() \
            and positions.device == dev, f"positions must be a contiguous int32 tensor {list(lead)} on {dev}"
    no_tangents("head_norm", q, k, q_weight, k_weight, cos, sin)
    if torch.is_grad_enabled():
        assert cos is None or not (cos.requires_grad or sin.requires_grad), "cos and sin have no gradient"
        if q.requires_grad or k.requires_grad or (q_weight is not None and q_weight.requires_grad) \
                or (k_weight is not None and k_weight.requires_grad):
            return _HeadNorm.apply(q, k, q_weight, k_weight, float(eps), positions, cos, sin)
    return _forward(q, k, q_weight, k_weight, float(eps), positions, cos, sin)[:2]

"""Matrix products grouped by expert, with a ragged number of rows for each.

``x [T, K]`` holds the rows sorted by expert: rows ``offsets[e] .. offsets[e + 1] - 1`` belong to expert e.  ``offsets`` is an int32 or
int64 device tensor ``[E + 1]`` that begins with 0, does not decrease and ends with T at most; it is read by the kernels
on the stream (no read-back: calls can be captured into graphs, and replayed with other offsets).  ``w [E, N, K]`` is dense, the contraction
index contiguous as in ``ops.head_gemm``; up to 512 experts, fewer than 2^29 rows, N and K up to 2^30.

    grouped_gemm        y[t, n] = sum_k x[t, k] w[e(t), n, k]             float16 / bfloat16, float32 sums, rounded once
    grouped_gemm_bwd    dx[t, k] = sum_n dy[t, n] w[e(t), n, k],  dw[e, n, k] = sum_{t in e} dy[t, n] x[t, k]
    grouped_fp8_gemm    the same product of e4m3 rows and block-128 e4m3 weights, every 128-channel block scaled in float32

Experts without rows cost nothing (their ``dw`` is zeros).  Rows behind the last expert's: zeros in an output made here, left as
they were in a caller-owned one, which must not overlap the operands (and makes a graph that has saved it refuse its backward pass).  Rows may have a pitch of their own; sizes of any kind are served, rows that begin on 16 bytes
by faster kernels.  ``grouped_gemm_apply`` is the differentiable form; a backward pass that is to be captured into a graph must not share its
leaves with an eager autograd graph that is still alive: capture ``grouped_gemm_bwd``, or drop the eager graph first.

The single-matrix sibling is ``nn/_tilelang/fused_fp8_gemm.py`` (operator caller ``FP8Linear.__call__``, cppmega_v4/nn/moe_fp8.py:89-93).
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import ops

__all__ = ["grouped_fp8_gemm", "grouped_gemm", "grouped_gemm_apply", "grouped_gemm_bwd"]


def _shape3(w: torch.Tensor, name: str) -> tuple[int, int, int]:
    if not isinstance(w, torch.Tensor) or w.ndim != 3:
        raise ValueError(f"{name} must be [E, N, K]; got {tuple(w.shape) if isinstance(w, torch.Tensor) else type(w).__name__}")
    return tuple(int(d) for d in w.shape)


def grouped_gemm(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """y [T, N] in x's type (a caller-owned ``out`` may be float32)."""
    if out is None:
        done = ops.host.grouped_gemm(x, w, offsets)
        if done is not None:
            return done
    fresh = out is None
    if fresh:
        out = torch.empty((x.shape[0], _shape3(w, "w")[1]), dtype=x.dtype, device=x.device)
    return ops.grouped_gemm(x, w, offsets, out=out, zero_tail=fresh)


def grouped_gemm_bwd(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, *, dx: torch.Tensor | None = None,
                     dw: torch.Tensor | None = None, need_dx: bool = True, need_dw: bool = True) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """``(dx [T, K], dw [E, N, K])`` in the operands' type (caller-owned ones may be float32); one that is not needed is None."""
    if dx is None and dw is None and need_dx and need_dw:
        done = ops.host.grouped_gemm_bwd(dy, x, w, offsets)
        if done is not None:
            return done
    E, N, K = _shape3(w, "w")
    if dy.ndim != 2 or x.ndim != 2 or tuple(dy.shape) != (x.shape[0], N) or x.shape[1] != K:
        raise ValueError(f"grouped_gemm_bwd shape mismatch: dy {tuple(dy.shape)}, x {tuple(x.shape)}, w {tuple(w.shape)}")
    if not (dy.dtype == x.dtype == w.dtype):
        raise TypeError(f"dy, x and w must have one type; got {dy.dtype}, {x.dtype}, {w.dtype}")
    fresh = dx is None
    if need_dx and fresh:
        dx = torch.empty((x.shape[0], K), dtype=x.dtype, device=x.device)
    if need_dw and dw is None:
        dw = torch.empty((E, N, K), dtype=w.dtype, device=w.device)
    elif need_dw and tuple(dw.shape) != (E, N, K):
        raise ValueError(f"dw must have shape {(E, N, K)}; got {tuple(dw.shape)}")
    if need_dx and need_dw:
        ops.grouped_gemm_backward(dy, x, w, offsets, dx=dx, dw=dw, zero_tail=fresh)
    elif need_dx:
        ops.grouped_gemm(dy, w, offsets, out=dx, zero_tail=fresh, transposed=True)
    elif need_dw:
        ops.grouped_weights_grad(dy, x, offsets, out=dw)
    return (dx if need_dx else None), (dw if need_dw else None)


def grouped_fp8_gemm(x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, offsets: torch.Tensor, *,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """y [T, N] in bfloat16 (or a caller-owned ``out``'s type: bfloat16, float16, float32).

    float16 and float32 results are sums of exact products; bfloat16 ones of many rows drop, of every eight products, what lies below
    2^-13 of the largest.

    ``x`` uint8 e4m3 [T, K] with float32 ``x_scale`` [T] or [T, ceil(K / 128)] (what ``rms_norm_fp8`` writes); ``w`` uint8 e4m3
    [E, N, K] with float32 ``w_scale`` [E, ceil(N / 128), ceil(K / 128)]."""
    if out is None:
        done = ops.host.grouped_fp8_gemm(x, x_scale, w, w_scale, offsets)
        if done is not None:
            return done
    fresh = out is None
    if fresh:
        out = torch.empty((x.shape[0], _shape3(w, "w")[1]), dtype=torch.bfloat16, device=x.device)
    return ops.grouped_fp8_gemm(x, x_scale, w, w_scale, offsets, out=out, zero_tail=fresh)


class _GroupedGemmFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, offsets):
        ctx.save_for_backward(x, w, offsets)
        return grouped_gemm(x, w, offsets)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, offsets = ctx.saved_tensors
        dy = dy if dy.is_contiguous() else dy.contiguous()
        dx, dw = grouped_gemm_bwd(dy, x, w, offsets, need_dx=ctx.needs_input_grad[0], need_dw=ctx.needs_input_grad[1])
        return dx, dw, None


def grouped_gemm_apply(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """Differentiable ``grouped_gemm``."""
    return _GroupedGemmFunction.apply(x, w, offsets)

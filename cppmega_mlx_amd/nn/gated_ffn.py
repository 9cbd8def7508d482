"""The gated feed-forward block: two projections, the activation and their product in one launch, with its gradients.

``x [T, K]`` holds rows, ``w [2 F, K]`` the gate's F rows and behind them the up projection's; the contraction index is contiguous, as in
``grouped_gemm``:

    g = x w_gate^T, u = x w_up^T        float32 sums of exact products
    gated_gemm       y = act(g) u       [T, F], rounded once
    gated_gemm_bwd   dg = dy u act'(g), du = dy act(g);  dx = dg w_gate + du w_up,  dw = (dg | du)^T x
    fp8_gated_gemm   the block of e4m3 rows and block-128 e4m3 weights

``activation``: "silu", g sigmoid(g); "gelu_tanh", 0.5 g (1 + tanh(sqrt(2 / pi) (g + 0.044715 g^3))).

By expert: ``w [E, 2 F, K]`` and ``offsets [E + 1]``, an int32 or int64 device tensor as ``grouped_gemm`` takes it (rows sorted by expert; read on
the stream, so that a captured call can be replayed with others; up to 512 experts).  Rows behind the last expert's: zeros in an output
made here, left as they were in a caller-owned one, which must not overlap the operands or another output (and makes a graph that has saved it
refuse its backward pass).  Rows may have a pitch of their own; fewer than 2^29 rows, F up to 2^29, K up to 2^30, and a launch of fewer than 2^32 threads (few rows
to an expert have 256 for 16 of its rows, whether they are there or not, and 32 outputs: more are refused); rows that begin on 16 bytes take the faster kernels.

The down projection behind the block is ``grouped_gemm`` (a dense one: ``grouped_gemm`` of one expert); for single tokens over 4-bit
weights see ``w4_gemm.py``.  A backward pass that is to be captured into a graph must not share its leaves with an eager autograd graph that is
still alive: capture ``gated_gemm_bwd``, or drop the eager graph first.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import ops

__all__ = ["fp8_gated_gemm", "gated_gemm", "gated_gemm_apply", "gated_gemm_bwd"]


def _outputs(w: torch.Tensor, offsets: torch.Tensor | None) -> int:
    if not isinstance(w, torch.Tensor) or w.ndim != (2 if offsets is None else 3) or w.shape[-2] % 2:
        shape = tuple(w.shape) if isinstance(w, torch.Tensor) else type(w).__name__
        raise ValueError(f"w must be {'[2 F, K] without offsets' if offsets is None else '[E, 2 F, K]'}; got {shape}")
    return int(w.shape[-2]) // 2


def gated_gemm(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor | None = None, *, activation: str = "silu", out: torch.Tensor | None = None,
               pre: torch.Tensor | None = None) -> torch.Tensor:
    """y [T, F] in x's type (a caller-owned ``out`` may be float32); caller-owned ``pre`` [T, 2 F], x's type or float32, takes g and u for
    the backward pass (rows behind the last expert are left alone)."""
    if out is None:
        done = ops.host.gated_gemm(x, w, offsets, ops.gate_code(activation), pre)
        if done is not None:
            return done
    fresh = out is None
    if fresh:
        out = torch.empty((x.shape[0], _outputs(w, offsets)), dtype=x.dtype, device=x.device)
    return ops.gated_gemm(x, w, offsets, activation=activation, out=out, pre=pre, zero_tail=fresh)


def gated_gemm_bwd(dy: torch.Tensor, pre: torch.Tensor, x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor | None = None, *,
                   activation: str = "silu", dx: torch.Tensor | None = None, dw: torch.Tensor | None = None, need_dx: bool = True,
                   need_dw: bool = True) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """``(dx [T, K], dw like w)`` in the operands' type (caller-owned ones may be float32); one that is not needed is None.

    dg and du are rounded to the operands' type between the two launches.  In float16 they are infinite from 65520 on (dx of that row and dw of
    that output are infinite or NaN then) and multiples of 2^-24 below 2^-14, whatever type the results have: scale the loss."""
    if dx is None and dw is None and need_dx and need_dw:
        done = ops.host.gated_gemm_bwd(dy, pre, x, w, offsets, ops.gate_code(activation))
        if done is not None:
            return done
    _outputs(w, offsets)
    fresh = dx is None
    if need_dx and fresh:
        dx = torch.empty((x.shape[0], x.shape[-1]), dtype=x.dtype, device=x.device)
    if need_dw and dw is None:
        dw = torch.empty(w.shape, dtype=w.dtype, device=w.device)
    dx, dw = dx if need_dx else None, dw if need_dw else None
    ops.gated_gemm_backward(dy, pre, x, w, offsets, activation=activation, dx=dx, dw=dw, zero_tail=fresh)
    return dx, dw


def fp8_gated_gemm(x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, offsets: torch.Tensor | None = None, *,
                   activation: str = "silu", out: torch.Tensor | None = None) -> torch.Tensor:
    """y [T, F] in bfloat16 (or a caller-owned ``out``'s type: bfloat16, float16, float32).

    ``x`` uint8 e4m3 [T, K] with float32 ``x_scale`` [T] or [T, ceil(K / 128)] (what ``rms_norm_fp8`` writes); ``w`` uint8 e4m3 [E, 2 F, K] with
    float32 ``w_scale`` [E, 2, ceil(F / 128), ceil(K / 128)]: either half has blocks of its own (without offsets no leading axis).
    float16 and float32 results come from sums of exact products; bfloat16 ones of many rows drop, of every eight products, what lies below
    2^-13 of the largest."""
    if out is None:
        done = ops.host.fp8_gated_gemm(x, x_scale, w, w_scale, offsets, ops.gate_code(activation))
        if done is not None:
            return done
    if not isinstance(x, torch.Tensor) or x.dtype != torch.uint8:
        raise TypeError(f"x must be 2D uint8 (fp8 storage); got {x.dtype if isinstance(x, torch.Tensor) else type(x).__name__}")
    fresh = out is None
    if fresh:
        out = torch.empty((x.shape[0], _outputs(w, offsets)), dtype=torch.bfloat16, device=x.device)
    return ops.gated_gemm(x, w, offsets, activation=activation, out=out, x_scale=x_scale, w_scale=w_scale, zero_tail=fresh)


class _GatedGemmFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, offsets, activation, pre_dtype, keep):
        if not keep:
            return gated_gemm(x, w, offsets, activation=activation)
        pre = torch.empty((x.shape[0], w.shape[-2]), dtype=pre_dtype, device=x.device)
        y = gated_gemm(x, w, offsets, activation=activation, pre=pre)
        ctx.save_for_backward(x, w, offsets, pre)
        ctx.activation = activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, offsets, pre = ctx.saved_tensors
        dy = dy if dy.is_contiguous() else dy.contiguous()
        dx, dw = gated_gemm_bwd(dy, pre, x, w, offsets, activation=ctx.activation, need_dx=ctx.needs_input_grad[0], need_dw=ctx.needs_input_grad[1])
        return dx, dw, None, None, None, None


def gated_gemm_apply(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor | None = None, *, activation: str = "silu",
                     pre_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Differentiable ``gated_gemm``: first derivatives, by the backward pass (a tangent of forward mode is refused).

    ``pre_dtype``: what the two products are kept in for the backward pass, float32 (unrounded) or x's type (half the memory; the
    gradients' error grows by a fifth, as one more rounding of theirs, and products beyond 65504 are infinite in float16).  They are not kept where no gradient is wanted."""
    # (by the function in either case: it refuses the derivatives that it lacks, where the bare call would drop them)
    return _GatedGemmFunction.apply(x, w, offsets, activation, pre_dtype, torch.is_grad_enabled() and (x.requires_grad or w.requires_grad))

"""RMS norm of the residual stream, with the residual's addition and 8-bit output.

    h = round(x + residual)                     the stream as stored, in the rows' type (x itself without a residual)
    y = h / sqrt(mean(h^2) + eps) * weight      in float32, rounded once

Rows are ``x[..., n]`` in float32 / float16 / bfloat16, n up to 32768, with a row pitch of their own; ``weight`` is ``[n]`` in the
rows' type or float32.  Outputs may be caller-owned: ``out`` may be ``x``, ``residual_out`` may be ``x`` or ``residual``; otherwise they
must not overlap what the call reads.  Writing into a tensor that autograd has saved makes that graph refuse its backward pass.

A row of zeros gives zeros for ``eps > 0``, a row with a NaN is NaN throughout; with an infinity it is NaN in that channel and zeros in the
others.  Squares and their sum are float32: a row whose sum leaves its range (a root mean square beyond 1.8e19 / sqrt(n)) gives zeros, and
``eps`` has to carry rows below 1e-19.

``rms_norm_fp8`` writes e4m3 codes and float32 scales in the layouts of ``SparseFP8KVCache`` and the FP8 projections:
one scale a row (``scale_block=0``) or per 128 channels (``scale_block=128``, the last block may be shorter), the codes taken from
the float32 values.  A row with a NaN has NaN codes throughout, beside scales of 1e-12
(1 with ``pow2_scales``).  ``rms_norm_bwd`` gives the gradients of the rows and of the weight, ``rms_norm_apply`` is the
differentiable form.  A backward pass that is to be captured into a graph must not share its leaves with an eager autograd graph
that is still alive (torch then synchronises with the eager stream inside the capture); capture ``rms_norm_bwd``, or drop
the eager graph first.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import ops

__all__ = ["rms_norm", "rms_norm_apply", "rms_norm_bwd", "rms_norm_fp8"]


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6, residual: torch.Tensor | None = None,
             out: torch.Tensor | None = None, residual_out: torch.Tensor | None = None) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """``y``, or ``(y, h)`` with a residual."""
    if out is None and residual_out is None:
        done = ops.host.rms_norm(x, weight, residual, eps, False, 0, False)
        if done is not None:
            return done
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if residual is not None and residual_out is None:
        residual_out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    ops.rms_norm(x, weight, eps=eps, out=out, residual=residual, residual_out=residual_out)
    return out if residual is None else (out, residual_out)


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6, residual: torch.Tensor | None = None, scale_block: int = 0,
                 pow2_scales: bool = False, codes: torch.Tensor | None = None, scale: torch.Tensor | None = None,
                 residual_out: torch.Tensor | None = None) -> tuple[torch.Tensor, ...]:
    """``(codes, scale)``, or ``(codes, scale, h)`` with a residual."""
    if codes is None and scale is None and residual_out is None:
        done = ops.host.rms_norm(x, weight, residual, eps, True, scale_block, bool(pow2_scales))
        if done is not None:
            return done
    if codes is None:
        codes = torch.empty(x.shape, dtype=torch.uint8, device=x.device)
    if scale is None:
        blocks = ((x.shape[-1] + 127) // 128,) if scale_block else ()
        scale = torch.empty(tuple(x.shape[:-1]) + blocks, dtype=torch.float32, device=x.device)
    if residual is not None and residual_out is None:
        residual_out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if codes.dtype != torch.uint8:
        raise TypeError(f"codes must be uint8 (fp8 storage); got {codes.dtype}")
    ops.rms_norm(x, weight, eps=eps, out=codes, residual=residual, residual_out=residual_out, scale=scale, scale_block=scale_block,
                 pow2_scales=pow2_scales)
    return (codes, scale) if residual is None else (codes, scale, residual_out)


def rms_norm_bwd(dy: torch.Tensor, h: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6, dh: torch.Tensor | None = None,
                 dx: torch.Tensor | None = None, dweight: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(dx, dweight)`` for the rows ``h`` that were normalised: ``dx`` (in h's type; of x and of the residual alike) includes
    ``dh``, the gradient that reaches the stream past the norm; ``dweight`` is float32, added in the same order on every run."""
    if dx is None and dweight is None:
        done = ops.host.rms_norm_bwd(dy, h, weight, eps, dh)
        if done is not None:
            return done
    if dx is None:
        dx = torch.empty(h.shape, dtype=h.dtype, device=h.device)
    if dweight is None:
        dweight = torch.empty((h.shape[-1],), dtype=torch.float32, device=h.device)
    ops.rms_norm_backward(dy, h, weight, eps=eps, dx=dx, dweight=dweight, dh=dh)
    return dx, dweight


def _dense(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() else t.contiguous()


class _RmsNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        ctx.set_materialize_grads(False)
        ctx.eps, ctx.with_residual = eps, residual is not None
        x = _dense(x)
        if residual is None:
            ctx.save_for_backward(x, weight)
            return rms_norm(x, weight, eps=eps)
        y, h = rms_norm(x, weight, eps=eps, residual=_dense(residual))
        ctx.save_for_backward(h, weight)
        return y, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight = ctx.saved_tensors
        if dy is None:                                   # only the stream was used
            return dh, None, dh, None
        dx, dweight = rms_norm_bwd(_dense(dy), h, weight, eps=ctx.eps, dh=None if dh is None else _dense(dh))
        return dx, dweight.to(weight.dtype), dx if ctx.with_residual else None, None


def rms_norm_apply(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *,
                   eps: float = 1e-6) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Differentiable ``rms_norm``: ``y``, or ``(y, h)`` with a residual."""
    return _RmsNormFunction.apply(x, weight, residual, float(eps))

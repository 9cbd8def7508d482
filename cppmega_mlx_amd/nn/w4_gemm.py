"""Products of few rows with 4-bit weights and group scales, plain or as the gated feed-forward block, dense or by expert.

``w [N, K / 2]`` uint8 holds two codes q = 0 .. 15 a byte, the even channel in the low four bits; ``scale`` (and ``bias``) ``[N, K / G]`` belong to
groups of G = 32, 64 or 128 channels, in x's type or float32:

    w4_gemm         y[t, n] = sum_k x[t, k] (scale[n, k / G] q[n, k] + bias[n, k / G]);  without biases scale (q - 8)
    w4_gated_gemm   act(x w_gate^T) (x w_up^T) over weights of 2 F rows, the gate's first

These are the bytes that an affine 4-bit quantiser packs into little-endian 32-bit words, eight channels a word (view those as uint8).  ``x [T, K]``
float16 or bfloat16, rows of any pitch; products are exact, sums float32, rounded once.  The codes enter as 16 + q, and 16 times a
group's sum of x comes off again: rows with infinities give NaN, and 32 times a group's sum of magnitudes must be finite in float32.

Made for the rows of a decode step: the codes are widened once for every 16 rows of an expert (64 where there are many), so long prompts
cost as many passes.  By expert: a leading axis ``[E, ..]`` and ``offsets [E + 1]`` as
in ``grouped_gemm``.  Rows behind the last expert's: zeros in an output made here, left as they were in a caller-owned one, which must not overlap
the operands.  Fewer than 2^29 rows, up to 2^24 elements apart, N up to 2^30, K up to 2^24, up to 512 experts, and fewer than 2^32
threads across the outputs (of up to four rows 2^29 outputs or, gated, 2^28 come to that, of more twice as many: they are refused).

The 8-bit sibling is ``nn/_tilelang/fused_fp8_gemm.py``; the block over 16- and 8-bit weights ``gated_ffn.py``.
"""

from __future__ import annotations

import torch

from .. import ops

__all__ = ["w4_gated_gemm", "w4_gemm"]


def _run(x, w, scale, bias, offsets, activation, out):
    if out is None:
        done = ops.host.w4_gemm(x, w, scale, bias, offsets, -1 if activation is None else ops.gate_code(activation))
        if done is not None:
            return done
    fresh = out is None
    if fresh:
        if not isinstance(w, torch.Tensor) or w.ndim != (2 if offsets is None else 3):
            raise ValueError(f"w must be {'[N, K / 2] without offsets' if offsets is None else '[E, N, K / 2]'}")
        out = torch.empty((x.shape[0], w.shape[-2] // (1 if activation is None else 2)), dtype=x.dtype, device=x.device)
    return ops.w4_gemm(x, w, scale, bias, offsets, out=out, activation=activation, zero_tail=fresh)


def w4_gemm(x: torch.Tensor, w: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor | None = None, offsets: torch.Tensor | None = None, *,
            out: torch.Tensor | None = None) -> torch.Tensor:
    """y [T, N] in x's type (a caller-owned ``out`` may be float32)."""
    return _run(x, w, scale, bias, offsets, None, out)


def w4_gated_gemm(x: torch.Tensor, w: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor | None = None, offsets: torch.Tensor | None = None, *,
                  activation: str = "silu", out: torch.Tensor | None = None) -> torch.Tensor:
    """y [T, F] in x's type (a caller-owned ``out`` may be float32) from weights of 2 F rows; activations as in ``gated_gemm``."""
    ops.gate_code(activation)
    return _run(x, w, scale, bias, offsets, activation, out)

/*
 * cppmega_mi355_ffn.h -- the feed-forward layer: the gated block (two projections, the activation and their product) in 16 and 8
 * bits with its gradients, and products with 4-bit weights.
 *
 * Same library (libcppmega_mi355.so) and same conventions as cppmega_mi355.h and cppmega_mi355_layer.h: a struct that starts with
 * `struct_size` plus its size, int status codes, caller-owned outputs, work enqueued on `stream`, device pointers, no allocation.
 * Pitches are in elements, the last axis of every operand is contiguous.
 *
 * Rows belong to experts as in the grouped products: rows offsets[e] .. offsets[e+1] - 1 to expert e, offsets[0] = 0,
 * non-decreasing, offsets[experts] <= rows, read on the device (offsets that break this give unspecified values, but no access outside
 * the operands).  offsets NULL: one expert has all rows.  Rows of an output from offsets[experts] on are left as they
 * were, or zeroed with zero_tail.
 *
 * A launch has fewer than 2^32 threads: a call whose sizes are within the limits below but whose tiles are more is refused
 * (UNSUPPORTED) before anything is written.  The gated block has 256 threads for 16 rows of an expert and 32 outputs at the least, so
 * up to 16 rows of one matrix reach that with 2^29 outputs; the 4-bit products have 256 for 32 outputs (gated: 16) of up to four rows of one matrix,
 * for 64 (32) of more.
 */
#ifndef CPPMEGA_MI355_FFN_H_
#define CPPMEGA_MI355_FFN_H_

#include "cppmega_mi355_layer.h"

#ifdef __cplusplus
extern "C" {
#endif

/* act(g) = g sigmoid(z(g)):  SILU z = g;  GELU_TANH z = 2 sqrt(2 / pi) (g + 0.044715 g^3), which is 0.5 g (1 + tanh(z / 2)) */
enum { CPPMEGA_MI355_GATE_NONE = -1, CPPMEGA_MI355_GATE_SILU = 0, CPPMEGA_MI355_GATE_GELU_TANH = 1 };
#define CPPMEGA_MI355_GATED_MAX_OUTPUTS 536870912   /* n of a gated block (k: CPPMEGA_MI355_GROUPED_MAX_SIZE) */

/* ---- gated block ----------------------------------------------------------------------
 *   g[t, j] = sum_k x[t, k] w[e(t), j, k],  u[t, j] = sum_k x[t, k] w[e(t), n + j, k],  y[t, j] = act(g) u
 * Products are exact, sums and the activation float32, y is rounded once.  pre, if given, takes g and u: the
 * backward pass starts from them.  E4M3 operands: scales as in cppmega_mi355_grouped_gemm, those of the weights float32
 * [experts, 2, ceil(n / 128), ceil(k / 128)] (either half has blocks of its own); BF16 results of many rows come from the
 * matrix instruction for e4m3 with what it drops; no pre. */
typedef struct cppmega_mi355_gated_gemm_args {
  uint32_t struct_size;
  int32_t activation;         /* CPPMEGA_MI355_GATE_SILU / _GELU_TANH                        */
  const void* x;              /* [rows, k]                                                   */
  const void* w;              /* [experts, 2 n, k] dense: the gate's rows, then the up projection's */
  void* y;                    /* [rows, n]                                                   */
  void* pre;                  /* [rows, 2 n] = g, u, or NULL                                 */
  const void* offsets;        /* [experts + 1], or NULL (experts = 1)                        */
  const float* x_scale;       /* E4M3                                                        */
  const float* w_scale;       /* E4M3                                                        */
  int32_t x_dtype;            /* BF16 / F16 / E4M3; w alike                                  */
  int32_t y_dtype;            /* x_dtype or F32; E4M3 operands: BF16 / F16 / F32             */
  int32_t pre_dtype;          /* x_dtype or F32                                              */
  int32_t offsets_dtype;      /* I32 / I64                                                   */
  int64_t rows;               /* below 2^29                                                  */
  int64_t x_pitch, y_pitch, pre_pitch;
  int32_t experts, n, k;
  int32_t x_scale_block;      /* 0 or 128                                                    */
  int32_t zero_tail;          /* of y; pre's rows behind the experts are never written       */
  int32_t reserved;
} cppmega_mi355_gated_gemm_args_t;

int cppmega_mi355_gated_gemm(const cppmega_mi355_gated_gemm_args_t* args, size_t args_size, void* stream);

/* Gradients, s = sigmoid(z(g)):
 *   dg = dy u (s + g s (1 - s) z'(g)),  du = dy g s    (float32, rounded to `dtype` in the workspace)
 *   dx = dg w_gate + du w_up,  dw = (dg | du)^T x      (zeros for an expert without rows)
 * F16: a dg or du of magnitude 65520 or more is an infinity (and dx of its row, dw of its output infinite or NaN), one
 * below 2^-14 a multiple of 2^-24, whatever the results' types; scale the loss, as for any gradient in float16.
 * The workspace holds dg and du; it need not be initialised. */
typedef struct cppmega_mi355_gated_gemm_bwd_args {
  uint32_t struct_size;
  int32_t activation;
  const void* dy;             /* [rows, n]                                                   */
  const void* pre;            /* [rows, 2 n] of the forward call                             */
  const void* x;              /* [rows, k]                                                   */
  const void* w;              /* [experts, 2 n, k] dense                                     */
  void* dx;                   /* [rows, k], or NULL: not wanted                              */
  void* dw;                   /* [experts, 2 n, k] dense, or NULL: not wanted                */
  const void* offsets;        /* [experts + 1], or NULL (experts = 1)                        */
  int32_t dtype;              /* BF16 / F16 of dy, x and w                                   */
  int32_t pre_dtype;          /* dtype or F32                                                */
  int32_t dx_dtype, dw_dtype; /* dtype or F32                                                */
  int32_t offsets_dtype;      /* I32 / I64                                                   */
  int32_t zero_tail;          /* of dx                                                       */
  int64_t rows;
  int64_t dy_pitch, pre_pitch, x_pitch, dx_pitch;
  int32_t experts, n, k;
  int32_t reserved;
  void* workspace;
  size_t workspace_bytes;
} cppmega_mi355_gated_gemm_bwd_args_t;

int cppmega_mi355_gated_gemm_bwd_workspace_bytes(const cppmega_mi355_gated_gemm_bwd_args_t* args, size_t args_size, size_t* bytes);
int cppmega_mi355_gated_gemm_bwd(const cppmega_mi355_gated_gemm_bwd_args_t* args, size_t args_size, void* stream);

/* ---- products with 4-bit weights ---------------------------------------------------------
 *   y[t, j] = sum_k x[t, k] (scale[j, k / group] q[j, k] + bias[j, k / group]);  without biases scale (q - 8)
 * q is 0 .. 15, two to a byte, the even channel in the low four bits.  Products with 16 + q are exact, sums float32: what is
 * added and taken away again is 16 times the rows' sums, so rows with infinities give NaN.  `activation` NONE: the product;
 * otherwise the gated block over weights [experts, 2 n, ..] as above.  Made for few rows: the codes are widened once for
 * every 16 rows of an expert, or for 64 where there are many. */
#define CPPMEGA_MI355_W4_MAX_CHANNELS 16777216   /* of k, and of x_pitch */
typedef struct cppmega_mi355_w4_gemm_args {
  uint32_t struct_size;
  int32_t activation;         /* CPPMEGA_MI355_GATE_NONE, or a gate                          */
  const void* x;              /* [rows, k]                                                   */
  const void* w;              /* [experts, n (gated: 2 n), k / 2] bytes, dense               */
  const void* scale;          /* [experts, n (2 n), k / group], dense                        */
  const void* bias;           /* like scale, or NULL                                         */
  void* y;                    /* [rows, n]                                                   */
  const void* offsets;        /* [experts + 1], or NULL (experts = 1)                        */
  int32_t x_dtype;            /* BF16 / F16                                                  */
  int32_t y_dtype;            /* x_dtype or F32                                              */
  int32_t scale_dtype;        /* x_dtype or F32; bias alike                                  */
  int32_t offsets_dtype;      /* I32 / I64                                                   */
  int64_t rows;               /* below 2^29                                                  */
  int64_t x_pitch, y_pitch;
  int32_t experts, n, k;
  int32_t group;              /* 32, 64 or 128; k is a multiple of it                        */
  int32_t zero_tail;
  int32_t reserved;
} cppmega_mi355_w4_gemm_args_t;

int cppmega_mi355_w4_gemm(const cppmega_mi355_w4_gemm_args_t* args, size_t args_size, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* CPPMEGA_MI355_FFN_H_ */

/*
 * cppmega_mi355_layer.h -- the operators that stand behind the attention call in a layer: the RMS norm of the
 * residual stream and the matrix products grouped by expert.
 *
 * Same library (libcppmega_mi355.so) and same conventions as cppmega_mi355.h: a struct that starts with
 * `struct_size` plus its size, int status codes, caller-owned outputs, work enqueued on `stream`, device
 * pointers, no allocation.  Pitches are in elements, the last axis of every operand is contiguous.
 */
#ifndef CPPMEGA_MI355_LAYER_H_
#define CPPMEGA_MI355_LAYER_H_

#include "cppmega_mi355.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- RMS norm with the residual's addition --------------------------------------------
 *   h = round(x + residual)  (x if there is no residual; rounded to the rows' type: the stream as stored)
 *   y = h / sqrt(mean(h^2) + eps) * weight,  in 32 bits, rounded once to `out`
 * out_dtype E4M3: `scale` float32 per row (scale_block 0) or per 128 channels (scale_block 128, the last
 * block may be shorter): max(amax|y| / 448, 1e-12), or with pow2_scales the smallest power of two with
 * 448 * scale >= amax (1 for a block of zeros; infinite for an infinite amax); codes are y / scale rounded to
 * nearest even (a NaN gives a NaN code; a row with one has scales of 1e-12, or 1).  Rows may be up to
 * CPPMEGA_MI355_NORM_MAX_WIDTH wide.  out may be x, residual_out may be x or residual; otherwise outputs must not
 * overlap the inputs.  Squares and their sum are float32. */
#define CPPMEGA_MI355_NORM_MAX_WIDTH 32768
typedef struct cppmega_mi355_rms_norm_args {
  uint32_t struct_size;
  int32_t x_dtype;            /* F32 / F16 / BF16; residual and residual_out alike          */
  const void* x;              /* [rows, width]                                               */
  const void* residual;       /* [rows, width], or NULL                                      */
  const void* weight;         /* [width]                                                     */
  int32_t weight_dtype;       /* F32, or x_dtype                                             */
  int32_t out_dtype;          /* x_dtype, or E4M3                                            */
  void* out;                  /* [rows, width]                                               */
  void* residual_out;         /* [rows, width] = h, or NULL                                  */
  float* scale;               /* E4M3: [rows] or [rows, ceil(width / 128)], dense            */
  int64_t rows;
  int64_t x_pitch, residual_pitch, out_pitch, residual_out_pitch;
  int32_t width;
  float eps;
  int32_t scale_block;        /* 0 or 128                                                    */
  int32_t pow2_scales;
} cppmega_mi355_rms_norm_args_t;

int cppmega_mi355_rms_norm(const cppmega_mi355_rms_norm_args_t* args, size_t args_size, void* stream);

/* Gradients for the rows h that were normalised (s = 1 / sqrt(mean(h^2) + eps), g = dy):
 *   dx[j] = dh[j] + s g[j] w[j] - s^3 h[j] mean(g w h)      (the gradient of x and of the residual alike)
 *   dweight[j] = sum over rows of g[j] h[j] s               (float32, in a fixed order)
 * The workspace holds partial sums of dweight; it need not be initialised. */
typedef struct cppmega_mi355_rms_norm_bwd_args {
  uint32_t struct_size;
  int32_t dtype;              /* F32 / F16 / BF16 of dy, h, dh and dx                        */
  const void* dy;             /* [rows, width]                                               */
  const void* h;              /* [rows, width]                                               */
  const void* weight;         /* [width]                                                     */
  const void* dh;             /* [rows, width] gradient that reaches the stream past the norm, or NULL */
  void* dx;                   /* [rows, width]; may be dy or dh                              */
  float* dweight;             /* [width]                                                     */
  int32_t weight_dtype;       /* F32, or dtype                                               */
  int32_t width;
  int64_t rows;
  int64_t dy_pitch, h_pitch, dh_pitch, dx_pitch;
  float eps;
  int32_t reserved;
  void* workspace;
  size_t workspace_bytes;
} cppmega_mi355_rms_norm_bwd_args_t;

int cppmega_mi355_rms_norm_bwd_workspace_bytes(const cppmega_mi355_rms_norm_bwd_args_t* args, size_t args_size, size_t* bytes);
int cppmega_mi355_rms_norm_bwd(const cppmega_mi355_rms_norm_bwd_args_t* args, size_t args_size, void* stream);

/* ---- matrix products grouped by expert ---------------------------------------------------
 * Rows offsets[e] .. offsets[e+1] - 1 of the row operands belong to expert e; offsets[0] = 0, non-decreasing,
 * offsets[experts] <= rows.  (They are read on the device: offsets that break this give unspecified values,
 * but no access outside the operands.)
 *   ROWS          y[t, n] = sum_k x[t, k] w[e(t), n, k]
 *   ROWS_GRAD     y[t, k] = sum_n x[t, n] w[e(t), n, k]     (x = dL/dy: the gradient of the rows)
 *   WEIGHTS_GRAD  y[e, n, k] = sum_{t in e} x[t, n] w[t, k] (x = dL/dy, w = the rows; zeros for no rows)
 * Products are exact, sums float32, rounded once.  ROWS with E4M3 operands: x_scale float32 [rows]
 * (x_scale_block 0) or [rows, ceil(k / 128)] (128), w_scale float32 [experts, ceil(n / 128), ceil(k / 128)];
 * every 128-channel block's sum is scaled in float32.  BF16 results of many rows come from the matrix
 * instruction for e4m3, which adds eight products at a time and drops what lies below 2^-13 of the largest of
 * them (not of their sum: where large products cancel, small ones may be lost); F16 and F32 results, and BF16
 * ones of few rows, are sums of exact products.
 * Rows of y from offsets[experts] on are left as they were, or zeroed with zero_tail. */
enum { CPPMEGA_MI355_GROUPED_ROWS = 0, CPPMEGA_MI355_GROUPED_ROWS_GRAD = 1, CPPMEGA_MI355_GROUPED_WEIGHTS_GRAD = 2 };
#define CPPMEGA_MI355_GROUPED_MAX_EXPERTS 512
#define CPPMEGA_MI355_GROUPED_MAX_SIZE 1073741824   /* of n and of k */

typedef struct cppmega_mi355_grouped_gemm_args {
  uint32_t struct_size;
  int32_t op;                 /* CPPMEGA_MI355_GROUPED_*                                     */
  const void* x;
  const void* w;              /* [experts, n, k] dense; WEIGHTS_GRAD: [rows, k]              */
  void* y;                    /* WEIGHTS_GRAD: [experts, n, k] dense                         */
  const void* offsets;        /* [experts + 1]                                               */
  const float* x_scale;       /* E4M3                                                        */
  const float* w_scale;       /* E4M3                                                        */
  int32_t x_dtype;            /* BF16 / F16 / E4M3; w alike                                  */
  int32_t y_dtype;            /* x_dtype or F32; E4M3 operands: BF16 / F16 / F32             */
  int32_t offsets_dtype;      /* I32 / I64                                                   */
  int32_t x_scale_block;      /* 0 or 128                                                    */
  int64_t rows;               /* below 2^29                                                  */
  int64_t x_pitch;            /* elements between rows of x                                  */
  int64_t w_pitch;            /* WEIGHTS_GRAD: elements between rows of w                    */
  int64_t y_pitch;            /* ROWS, ROWS_GRAD: elements between rows of y                 */
  int32_t experts, n, k;
  int32_t zero_tail;
} cppmega_mi355_grouped_gemm_args_t;

int cppmega_mi355_grouped_gemm(const cppmega_mi355_grouped_gemm_args_t* args, size_t args_size, void* stream);

/* The calls of a ROWS_GRAD and a WEIGHTS_GRAD block (independent of each other), in one launch where their kernels allow it. */
int cppmega_mi355_grouped_gemm_bwd(const cppmega_mi355_grouped_gemm_args_t* rows, const cppmega_mi355_grouped_gemm_args_t* weights,
                                   size_t args_size, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* CPPMEGA_MI355_LAYER_H_ */

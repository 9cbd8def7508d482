// Gradients of the gated feed-forward block (gfx950): dg and du of every row from dy and the two products that the forward call kept, then
// dx and dw as one grouped product's two gradients over the 2 n rows of the weight.
//
// dg and du are rounded to the rows' type, as any gradient between two 16-bit products is: the matrix cores take nothing wider.  In float16 that
// bounds them: an infinity from 65520 on, steps of 2^-24 below 2^-14.  (A power of two taken off and put back needs the largest of all of them
// first, a second pass over dy, g and u: a scaled loss does the same for nothing.)
// Their kernel is bound by memory: of a row and output dy, g and u read and dg, du written once; of 8192 rows x 2048 outputs, behind
// the forward call (the last-level cache still has part of what it kept), 168 MB in 34 us, with float32 g and u 235 MB in 36.

#include <string.h>

#include "grouped_gemm.h"

namespace cm {

int grouped_gemm_launch_as(const char* call, const cppmega_mi355_grouped_gemm_args_t& a, hipStream_t stream);
int grouped_gemm_bwd_launch_as(const char* call, const cppmega_mi355_grouped_gemm_args_t& rows, const cppmega_mi355_grouped_gemm_args_t& weights, hipStream_t stream);
int grouped_gemm_check(const char* call, const cppmega_mi355_grouped_gemm_args_t& rows, const cppmega_mi355_grouped_gemm_args_t& weights, bool need_rows, bool need_weights);

namespace {

struct GradParams {
  const void *dy, *pre;
  unsigned short* grad;
  const void* offsets;
  long long rows, dy_pitch, pre_pitch, grad_pitch;
  int n, experts, offsets64, activation, f16, pre32;
};

constexpr int kThreads = 256, kRun = 8;                          // outputs of a thread

// As many of kRun 16-bit or float32 values as are there.
template <bool WHOLE>
__device__ __forceinline__ void load_run(const void* base, size_t at, int count, bool wide, bool f16, float (&v)[kRun]) {
  if (WHOLE && !wide) {
    u32x4 r;
    __builtin_memcpy(&r, (const unsigned short*)base + at, 16);
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const unsigned short b = (unsigned short)(r[i >> 1] >> (16 * (i & 1)));
      v[i] = f16 ? f16_bits_to_f32(b) : bf16_bits_to_f32(b);
    }
  } else if (WHOLE) {
    __builtin_memcpy(v, (const float*)base + at, 4 * kRun);
  } else {
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const int dtype = wide ? CPPMEGA_MI355_F32 : f16 ? CPPMEGA_MI355_F16 : CPPMEGA_MI355_BF16;
      v[i] = i < count ? load_as(base, at + i, dtype) : 0.0f;
    }
  }
}

template <bool WHOLE>
__device__ __forceinline__ void run_grads(const GradParams& p, long long row, int col) {
  const int count = p.n - col;
  float dy[kRun], g[kRun], u[kRun], dg[kRun], du[kRun];
  load_run<WHOLE>(p.dy, (size_t)row * p.dy_pitch + col, count, false, p.f16, dy);
  load_run<WHOLE>(p.pre, (size_t)row * p.pre_pitch + col, count, p.pre32, p.f16, g);
  load_run<WHOLE>(p.pre, (size_t)row * p.pre_pitch + p.n + col, count, p.pre32, p.f16, u);
#pragma unroll
  for (int i = 0; i < kRun; ++i) gate_grads(g[i], u[i], dy[i], p.activation, dg[i], du[i]);
  unsigned short* const at = p.grad + (size_t)row * p.grad_pitch + col;
  auto store = [&](unsigned short* to, const float (&v)[kRun]) {
    unsigned r[kRun / 2];
#pragma unroll
    for (int i = 0; i < kRun / 2; ++i) r[i] = p.f16 ? pack_f16(v[2 * i], v[2 * i + 1]) : pack_bf16(v[2 * i], v[2 * i + 1]);
    if (WHOLE) {
      __builtin_memcpy(to, r, 2 * kRun);
    } else {
#pragma unroll
      for (int i = 0; i < kRun; ++i)
        if (i < count) to[i] = (unsigned short)(r[i >> 1] >> (16 * (i & 1)));
    }
  };
  store(at, dg);
  store(at + p.n, du);
}

// One thread per run of a row, 2^log_across of them to a row in a block; rows behind the last expert are not touched (their gradients are never
// read).
__global__ __launch_bounds__(kThreads) void gated_grad_kernel(const GradParams p, const int log_across, const unsigned across_blocks) {
  const unsigned down = blockIdx.x / across_blocks, part = blockIdx.x - down * across_blocks;
  const long long row = ((long long)down << (8 - log_across)) + (threadIdx.x >> log_across);
  const int col = (int)((part << log_across) + (threadIdx.x & ((1u << log_across) - 1))) * kRun;
  long long last = p.rows;
  if (p.offsets) {
    const long long o = p.offsets64 ? ((const long long*)p.offsets)[p.experts] : (long long)((const int*)p.offsets)[p.experts];
    last = o < last ? o : last;
  }
  if (row >= last || col >= p.n) return;
  if (col + kRun <= p.n) run_grads<true>(p, row, col);
  else run_grads<false>(p, row, col);
}

// Elements between rows of dg | du: rows begin on 16 bytes.
long long grad_pitch(int n) { return (2ll * n + 7) / 8 * 8; }

}  // namespace

int gated_gemm_bwd_workspace_bytes(const cppmega_mi355_gated_gemm_bwd_args_t& a, size_t* bytes) {
  if (a.rows < 0 || a.rows > 0x1fffffffll || a.n < 1 || a.n > CPPMEGA_MI355_GATED_MAX_OUTPUTS)
    return fail(CPPMEGA_MI355_ERR_SHAPE, "gated_gemm_bwd: rows=%lld n=%d", (long long)a.rows, a.n);
  *bytes = (size_t)a.rows * grad_pitch(a.n) * 2;
  return 0;
}

int gated_gemm_bwd_launch(const cppmega_mi355_gated_gemm_bwd_args_t& a, hipStream_t stream) {
  size_t need = 0;
  if (int rc = gated_gemm_bwd_workspace_bytes(a, &need)) return rc;
  if (a.activation != CPPMEGA_MI355_GATE_SILU && a.activation != CPPMEGA_MI355_GATE_GELU_TANH)
    return fail(CPPMEGA_MI355_ERR_SHAPE, "gated_gemm_bwd: unknown activation %d", a.activation);
  if (a.dtype != CPPMEGA_MI355_F16 && a.dtype != CPPMEGA_MI355_BF16)
    return fail(CPPMEGA_MI355_ERR_DTYPE, "gated_gemm_bwd: operands of dtype %d are not float16 / bfloat16", a.dtype);
  if (a.pre_dtype != a.dtype && a.pre_dtype != CPPMEGA_MI355_F32)
    return fail(CPPMEGA_MI355_ERR_DTYPE, "gated_gemm_bwd: pre of dtype %d beside operands of dtype %d", a.pre_dtype, a.dtype);
  if (a.rows > 0 && (!a.dy || !a.pre)) return fail(CPPMEGA_MI355_ERR_NULL, "gated_gemm_bwd: dy / pre is NULL");
  if (!a.offsets && a.experts != 1) return fail(CPPMEGA_MI355_ERR_NULL, "gated_gemm_bwd: offsets is NULL");
  if (a.offsets && a.offsets_dtype != CPPMEGA_MI355_I32 && a.offsets_dtype != CPPMEGA_MI355_I64)
    return fail(CPPMEGA_MI355_ERR_DTYPE, "gated_gemm_bwd: offsets must be int32 or int64");
  if (!a.dx && !a.dw) return 0;
  if (need && (!a.workspace || a.workspace_bytes < need))
    return fail(CPPMEGA_MI355_ERR_WORKSPACE, "gated_gemm_bwd: a workspace of %zu bytes is needed, got %zu", need, a.workspace_bytes);
  if ((uintptr_t)a.workspace & 15) return fail(CPPMEGA_MI355_ERR_ALIGNMENT, "gated_gemm_bwd: the workspace must begin on 16 bytes");
  cppmega_mi355_grouped_gemm_args_t r;
  memset(&r, 0, sizeof(r));
  r.x_dtype = a.dtype; r.offsets_dtype = a.offsets ? a.offsets_dtype : CPPMEGA_MI355_I32; r.offsets = a.offsets;
  r.rows = a.rows; r.experts = a.experts; r.n = 2 * a.n; r.k = a.k;
  r.x = a.workspace; r.x_pitch = grad_pitch(a.n);
  cppmega_mi355_grouped_gemm_args_t w = r;
  r.op = kRowsGrad; r.w = a.w; r.y = a.dx; r.y_dtype = a.dx_dtype; r.y_pitch = a.dx_pitch; r.zero_tail = a.zero_tail;
  w.op = kWeightsGrad; w.w = a.x; w.w_pitch = a.x_pitch; w.y = a.dw; w.y_dtype = a.dw_dtype;
  if (a.rows > 0) {
    const int runs = (a.n + kRun - 1) / kRun;
    int log_across = 0;
    while (log_across < 8 && (1 << log_across) < runs) ++log_across;
    const long long across = (runs + (1 << log_across) - 1) >> log_across, blocks = across * (((a.rows << log_across) + kThreads - 1) / kThreads);
    if (int rc = check_tiles("gated_gemm_bwd", blocks, kThreads)) return rc;
    // (what the products refuse is refused before the first launch)
    if (int rc = grouped_gemm_check("gated_gemm_bwd", r, w, a.dx != nullptr, a.dw != nullptr)) return rc;
    GradParams p;
    p.dy = a.dy; p.pre = a.pre; p.grad = (unsigned short*)a.workspace; p.offsets = a.offsets;
    p.rows = a.rows; p.dy_pitch = a.dy_pitch; p.pre_pitch = a.pre_pitch; p.grad_pitch = grad_pitch(a.n);
    p.n = a.n; p.experts = a.experts; p.offsets64 = a.offsets_dtype == CPPMEGA_MI355_I64; p.activation = a.activation;
    p.f16 = a.dtype == CPPMEGA_MI355_F16; p.pre32 = a.pre_dtype == CPPMEGA_MI355_F32;
    hipLaunchKernelGGL(gated_grad_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, stream, p, log_across, (unsigned)across);
    CM_HIP_CHECK(hipGetLastError());
  }
  if (a.dx && a.dw) return grouped_gemm_bwd_launch_as("gated_gemm_bwd", r, w, stream);
  return grouped_gemm_launch_as("gated_gemm_bwd", a.dx ? r : w, stream);
}

}  // namespace cm

// Products grouped by expert for operands of any alignment, pitch and size (gfx950): odd row lengths, views whose rows do not begin on 16
// bytes, and float16 and float32 results of e4m3 operands (as bfloat16, whose products are exact).  The aligned kernels let the load unit write to LDS,
// which wants whole 16-byte pieces; here a piece goes through registers, by one (unaligned) load where it is whole and element by element
// at the end of a row.  Bound by those loads: a step's wait for the one before it.  Measured, 16384 rows of 32 experts, 4096 x 2049 bf16:
// 597 us (461 TFLOP/s; 2048: 313 by the aligned tiles), both gradients 1610; 4097 x 2048, whose forward the tiles take (326), both gradients 1315;
// e4m3 into float16 or float32, 4096 x 2048: 642 (into bfloat16 164).
//
// One workgroup of four wavefronts per 128 x 128 tile, 128 bytes of contraction a step (one scale block of e4m3), the next
// step's pieces on their way under the products of this one.  Pieces are 16 bytes; in LDS
//   contraction contiguous: [row][8 pieces], piece c of row r in place c ^ (r / 2 % 8): sixteen rows with one piece lie in different
//     banks;
//   contraction slow: [step of 64][16 pieces of 8 channels], piece c of step s in place c ^ 4 (s % 4): the four rows of a transposing
//     read lie in different banks.

#include "grouped_gemm.h"

namespace cm {
namespace {

constexpr int BM = 128, BN = 128;

template <int BYTES>
struct Code { typedef unsigned short type; };
template <>
struct Code<1> { typedef unsigned char type; };

template <int BYTES>
__device__ __forceinline__ u32x4 piece(const char* at, long long valid) {     // elements of the piece that exist
  typedef typename Code<BYTES>::type T;
  u32x4 r = {0u, 0u, 0u, 0u};
  if (valid >= 16 / BYTES) {
    __builtin_memcpy(&r, at, 16);
  } else if (valid > 0) {
    T e[16 / BYTES];
#pragma unroll
    for (int i = 0; i < 16 / BYTES; ++i) e[i] = i < valid ? ((const T*)at)[i] : (T)0;
    __builtin_memcpy(&r, e, 16);
  }
  return r;
}

template <int OP, int DT>
__global__ __launch_bounds__(256) void grouped_general_kernel(const GroupedParams p) {
  constexpr bool FP8 = DT == CPPMEGA_MI355_E4M3, F16 = DT == CPPMEGA_MI355_F16;
  constexpr int BYTES = FP8 ? 1 : 2, STEP = 128 / BYTES;            // elements of contraction in a step
  constexpr bool TR = OP == kWeightsGrad, TQ = OP != kRows;         // the contraction is the operand's slow axis
  __shared__ u32x4 lr[BM * 8], lq[BN * 8];
  __shared__ int starts[kMaxExperts + 2];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int l32 = lane & 31, half = lane >> 5;

  // ---- which tile ----
  const int rows_c = OP == kWeightsGrad ? p.n : 0, cols_c = OP == kRows ? p.n : p.k;
  const int tiles_n = (cols_c + BN - 1) / BN;
  int e, m0, n0;
  long long lo, hi;
  if (OP == kWeightsGrad) {
    const int per = ((rows_c + BM - 1) / BM) * tiles_n;
    e = (int)blockIdx.x / per;
    const int t = (int)blockIdx.x - e * per;
    m0 = t / tiles_n * BM;
    n0 = t % tiles_n * BN;
    lo = offset_of(p, e);
    hi = offset_of(p, e + 1);
  } else {
    const int total = fill_tiles<BM>(p, starts);
    const int mt = (int)(blockIdx.x / (unsigned)tiles_n);
    if (mt >= total) return;
    e = expert_of_tile(p, starts, mt);
    lo = offset_of(p, e);
    hi = e < p.experts ? offset_of(p, e + 1) : p.rows;
    m0 = (mt - starts[e]) * BM;
    n0 = (int)(blockIdx.x % (unsigned)tiles_n) * BN;
  }
  const long long tokens = hi > lo ? hi - lo : 0;
  const long long contraction = OP == kWeightsGrad ? tokens : (e == p.experts ? 0 : (OP == kRows ? p.k : p.n));
  const long long rows_here = (OP == kWeightsGrad ? rows_c : tokens) - m0;          // rows of C from m0 on
  const long long cols_here = cols_c - n0;
  const size_t weight = (size_t)e * p.n * p.k;
  const char* const xb = (const char*)p.x + (size_t)lo * p.x_pitch * BYTES;
  const char* const wb = (const char*)p.w + (OP == kWeightsGrad ? (size_t)lo * p.w_pitch : e < p.experts ? weight : 0) * BYTES;
  const long long w_pitch = OP == kWeightsGrad ? p.w_pitch : p.k;

  // a thread's four pieces of each operand
  u32x4 pr[4], pq[4];
  auto fetch = [&](bool transposed, const char* base, long long pitch, int first, long long here, long long k0, u32x4 (&to)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int u = i * 256 + tid;
      if (!transposed) {
        const int row = u >> 3, c = u & 7;
        const long long k = k0 + c * (16 / BYTES);
        to[i] = piece<BYTES>(base + ((first + row) * pitch + k) * BYTES, row < here ? contraction - k : 0);
      } else {
        const int step = u >> 4, c = u & 15;
        to[i] = piece<BYTES>(base + ((k0 + step) * pitch + first + c * 8) * BYTES, k0 + step < contraction ? here - c * 8 : 0);
      }
    }
  };
  auto keep = [&](bool transposed, u32x4* lds, const u32x4 (&from)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int u = i * 256 + tid;
      if (!transposed) lds[(u >> 3) * 8 + ((u & 7) ^ ((u >> 4) & 7))] = from[i];
      else lds[(u >> 4) * 16 + ((u & 15) ^ (((u >> 4) & 3) << 2))] = from[i];
    }
  };
  // 32 rows (or columns) from `at` on, 16 steps (16 bits) of contraction: lane l holds row l % 32, steps 8 (l / 32) ..
  auto operand16 = [&](bool transposed, const u32x4* lds, int at, int ks) -> bf16x8 {
    if (!transposed) {
      const int row = at + l32;
      return __builtin_bit_cast(bf16x8, lds[row * 8 + ((2 * ks + half) ^ ((row >> 1) & 7))]);
    }
    const int l16 = lane & 15, col = at + (lane & 16) + (l16 & 3) * 4;
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    u32x4 r;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int step = ks * 16 + half * 8 + j * 4 + (l16 >> 2);
      const char* a = (const char*)lds + (step * 16 + ((col >> 3) ^ ((step & 3) << 2))) * 16 + (col & 4) * 2;
      const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)a));
      r[2 * j] = v[0];
      r[2 * j + 1] = v[1];
    }
    return __builtin_bit_cast(bf16x8, r);
  };
  // a wavefront has 64 x 64 of the tile; the columns of C are the first operand, so that a lane holds runs of 4 of them
  const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
  f32x16 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.0f;
  const int blocks_k = (p.k + 127) / 128;
  const long long steps = (contraction + STEP - 1) / STEP;
  if (steps > 0) {
    fetch(TR, xb, p.x_pitch, m0, rows_here, 0, pr);
    fetch(TQ, wb, w_pitch, n0, cols_here, 0, pq);
  }
  for (long long s = 0; s < steps; ++s) {
    __syncthreads();
    keep(TR, lr, pr);
    keep(TQ, lq, pq);
    __syncthreads();
    if (s + 1 < steps) {
      fetch(TR, xb, p.x_pitch, m0, rows_here, (s + 1) * STEP, pr);
      fetch(TQ, wb, w_pitch, n0, cols_here, (s + 1) * STEP, pq);
    }
    if constexpr (FP8) {
      float sx[2], sw;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const long long row = m0 + wm + i * 32 + l32;
        sx[i] = row < tokens ? p.x_scale[p.x_scale_block ? (size_t)(lo + row) * blocks_k + s : (size_t)(lo + row)] : 0.0f;
      }
      sw = n0 < p.n ? p.w_scale[((size_t)e * ((p.n + 127) / 128) + n0 / 128) * blocks_k + s] : 0.0f;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          f32x16 t;
#pragma unroll
          for (int v = 0; v < 16; ++v) t[v] = 0.0f;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            // 16 codes of a row as two operands of 16 bits: exact, where the matrix instruction for codes would drop low bits
            const int rq = wn + j * 32 + l32, rr = wm + i * 32 + l32;
            const u32x4 q = lq[rq * 8 + ((2 * c + half) ^ ((rq >> 1) & 7))], r = lr[rr * 8 + ((2 * c + half) ^ ((rr >> 1) & 7))];
            t = __builtin_amdgcn_mfma_f32_32x32x16_bf16(cvt8(q[0], q[1]), cvt8(r[0], r[1]), t, 0, 0, 0);
            t = __builtin_amdgcn_mfma_f32_32x32x16_bf16(cvt8(q[2], q[3]), cvt8(r[2], r[3]), t, 0, 0, 0);
          }
          const float f = sx[i] * sw;
#pragma unroll
          for (int v = 0; v < 16; ++v) acc[i][j][v] = fmaf(f, t[v], acc[i][j][v]);
        }
    } else {
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        bf16x8 a[2], b[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) a[j] = operand16(TQ, lq, wn + j * 32, ks);
#pragma unroll
        for (int i = 0; i < 2; ++i) b[i] = operand16(TR, lr, wm + i * 32, ks);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            if constexpr (F16) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a[j]), __builtin_bit_cast(f16x8, b[i]), acc[i][j], 0, 0, 0);
            else acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[j], b[i], acc[i][j], 0, 0, 0);
          }
      }
    }
  }
  // lane: row l % 32 of the tile, columns 8 q + 4 (l / 32) + 0..3
  const size_t row0 = OP == kWeightsGrad ? (size_t)e * p.n + m0 : (size_t)lo + m0;
  const long long y_pitch = OP == kWeightsGrad ? p.k : p.y_pitch;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = wm + i * 32 + l32;
    if (row >= rows_here) continue;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const int col = wn + j * 32 + (v >> 2) * 8 + half * 4 + (v & 3);
        if (col < cols_here) store_as(p.y, (row0 + row) * y_pitch + n0 + col, p.y_dtype, acc[i][j][v]);
      }
  }
}

}  // namespace

int grouped_general_launch(const GroupedParams& p, int op, int dtype, hipStream_t stream) {
  const long long tiles_n = ((op == kRows ? p.n : p.k) + BN - 1) / BN;
  const long long tiles_m = op == kWeightsGrad ? (long long)p.experts * ((p.n + BM - 1) / BM) : p.rows / BM + p.experts + 1;
  if (int rc = check_tiles(tiles_m * tiles_n, 256)) return rc;
  const dim3 grid((unsigned)(tiles_m * tiles_n)), block(256);
#define CM_GENERAL(op_, dt) hipLaunchKernelGGL((grouped_general_kernel<op_, dt>), grid, block, 0, stream, p)
#define CM_GENERAL_OP(op_)                                           \
  do {                                                               \
    if (dtype == CPPMEGA_MI355_F16) CM_GENERAL(op_, CPPMEGA_MI355_F16); \
    else CM_GENERAL(op_, CPPMEGA_MI355_BF16);                        \
  } while (0)
  if (dtype == CPPMEGA_MI355_E4M3) CM_GENERAL(kRows, CPPMEGA_MI355_E4M3);
  else if (op == kRows) CM_GENERAL_OP(kRows);
  else if (op == kRowsGrad) CM_GENERAL_OP(kRowsGrad);
  else CM_GENERAL_OP(kWeightsGrad);
#undef CM_GENERAL_OP
#undef CM_GENERAL
  CM_HIP_CHECK(hipGetLastError());
  return 0;
}

}  // namespace cm

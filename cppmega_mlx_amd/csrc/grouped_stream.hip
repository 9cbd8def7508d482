// Products grouped by expert for few rows (gfx950): the experts' weights pass once, straight into registers.
//
// Bound by memory: an expert with 16 rows has 16 products for every weight byte pair that it reads, the matrix cores could do two
// hundred.  A workgroup has 16 TM rows of one expert and 16 TN outputs; its four wavefronts divide the contraction, and their sums meet in LDS
// once at the end, added in order.  A step is 128 bytes of every weight row (whole cache lines), requested one step ahead; the
// activations' pieces come from the caches, 1 / TN of the traffic.  Which expert a workgroup has, every wavefront finds by itself
// (a scan over the counts in registers: no table, no barrier in front of the first load).
//
// e4m3 codes become bfloat16 on the way, which is exact; a step is one 128-channel block, whose sum is scaled in float32.

#include "grouped_gemm.h"

namespace cm {
namespace {

constexpr int kWaves = 4;

template <int DT, int TM, int TN>
__global__ __launch_bounds__(64 * kWaves, 2) void grouped_stream_kernel(const GroupedParams p) {
  constexpr bool FP8 = DT == CPPMEGA_MI355_E4M3, F16 = DT == CPPMEGA_MI355_F16;
  constexpr int BYTES = FP8 ? 1 : 2, STEP = 128 / BYTES, BM = 16 * TM, BN = 16 * TN;
  __shared__ f32x4 sums[kWaves][TM * TN][64];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int l16 = lane & 15, quad = lane >> 4;

  // ---- which tile ----
  const int tiles_n = (p.n + BN - 1) / BN;
  const int mt = (int)(blockIdx.x / (unsigned)tiles_n), n0 = (int)(blockIdx.x % (unsigned)tiles_n) * BN;
  int e = -1, first = 0, rows = 0;
  for (int e0 = 0, before = 0; e0 <= p.experts; e0 += 64) {
    const int x = e0 + lane;
    int lo = 0, count = 0;
    if (x <= p.experts) {                                        // (the last entry: rows behind the experts, to be zeroed)
      lo = (int)offset_of(p, x);
      const int hi = x < p.experts ? (int)offset_of(p, x + 1) : (p.zero_tail ? (int)p.rows : lo);
      count = hi > lo ? hi - lo : 0;
    }
    const int tiles = (count + BM - 1) / BM, through = before + (int)wave_inclusive_sum_dpp((unsigned)tiles);
    const unsigned long long behind = __ballot(through > mt);
    if (behind) {
      const int at = (int)__builtin_ctzll(behind);
      const int m0 = (mt - (__builtin_amdgcn_readlane(through, at) - __builtin_amdgcn_readlane(tiles, at))) * BM;
      e = e0 + at;
      first = __builtin_amdgcn_readlane(lo, at) + m0;
      rows = __builtin_amdgcn_readlane(count, at) - m0;
      break;
    }
    before = __builtin_amdgcn_readlane(through, 63);
  }
  if (e < 0) return;

  // ---- this wavefront's steps ----
  const int steps = e < p.experts ? (p.k + STEP - 1) / STEP : 0;
  const int s0 = steps * wave / kWaves, s1 = steps * (wave + 1) / kWaves;
  const int blocks_k = (p.k + 127) / 128;
  const char *wat[TN], *xat[TM];
  const float* sxat[TM];
  const float* swat = nullptr;
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int n = n0 + j * 16 + l16;
    wat[j] = (const char*)p.w + ((size_t)(e < p.experts ? e : 0) * p.n + (n < p.n ? n : p.n - 1)) * p.k * BYTES + quad * 16;
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int row = i * 16 + l16;                                // (rows past the end repeat the last one and are not stored)
    const size_t at = (size_t)(first + (row < rows ? row : rows - 1));
    xat[i] = (const char*)p.x + at * p.x_pitch * BYTES + quad * 16;
    if (FP8) sxat[i] = p.x_scale + at * (p.x_scale_block ? blocks_k : 1);
  }
  if (FP8) swat = p.w_scale + ((size_t)(e < p.experts ? e : 0) * ((p.n + 127) / 128) + n0 / 128) * blocks_k;

  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  u32x4 w[2][TN][2], x[2][TM][2];
  float sx[2][TM], sw[2];
  auto load = [&](int s, int to) {
    const size_t at = (size_t)s * 128;
    const int left = p.k * BYTES - s * 128 - quad * 16;          // bytes of the row from this lane's piece on
    const bool there[2] = {left > 0, left > 64};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int j = 0; j < TN; ++j) w[to][j][h] = there[h] ? __builtin_nontemporal_load((const u32x4*)(wat[j] + at + h * 64)) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
      for (int i = 0; i < TM; ++i)
        if (i == 0 || i * 16 < rows) x[to][i][h] = there[h] ? *(const u32x4*)(xat[i] + at + h * 64) : u32x4{0u, 0u, 0u, 0u};
    }
    if (FP8) {
#pragma unroll
      for (int i = 0; i < TM; ++i)
        if (i == 0 || i * 16 < rows) sx[to][i] = sxat[i][p.x_scale_block ? s : 0];
      sw[to] = swat[s];
    }
  };
  auto multiply = [&](int b) {
    if constexpr (FP8) {
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        f32x4 t[TM];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const bf16x8 wv = cvt8(w[b][j][h][2 * c], w[b][j][h][2 * c + 1]);
#pragma unroll
            for (int i = 0; i < TM; ++i)
              if (i == 0 || i * 16 < rows)
                t[i] = mm<false>(wv, cvt8(x[b][i][h][2 * c], x[b][i][h][2 * c + 1]), h + c == 0 ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : t[i]);
          }
#pragma unroll
        for (int i = 0; i < TM; ++i)
          if (i == 0 || i * 16 < rows) {
            const float f = sx[b][i] * sw[b];
#pragma unroll
            for (int v = 0; v < 4; ++v) acc[i][j][v] = fmaf(f, t[i][v], acc[i][j][v]);
          }
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < TM; ++i)
          if (i == 0 || i * 16 < rows) {
#pragma unroll
            for (int j = 0; j < TN; ++j)
              acc[i][j] = mm<F16>(__builtin_bit_cast(bf16x8, w[b][j][h]), __builtin_bit_cast(bf16x8, x[b][i][h]), acc[i][j]);
          }
    }
  };
  if (s0 < s1) load(s0, 0);
  for (int s = s0; s < s1; s += 2) {
    if (s + 1 < s1) load(s + 1, 1);
    multiply(0);
    if (s + 1 < s1) {
      if (s + 2 < s1) load(s + 2, 0);
      multiply(1);
    }
  }
  // ---- the wavefronts' sums, in order; lane: row l % 16, outputs 4 (l / 16) + 0..3 of a tile ----
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) sums[wave][i * TN + j][lane] = acc[i][j];
  __syncthreads();
#pragma unroll
  for (int u0 = 0; u0 < TM * TN; u0 += kWaves) {
    const int u = u0 + wave;
    if (u >= TM * TN) break;
    f32x4 v = sums[0][u][lane];
#pragma unroll
    for (int k = 1; k < kWaves; ++k) v += sums[k][u][lane];
    const int row = u / TN * 16 + l16, n = n0 + u % TN * 16 + quad * 4;
    if (row >= rows || n >= p.n) continue;
    const size_t at = (size_t)(first + row) * p.y_pitch + n;
    if (n + 4 <= p.n && p.y_dtype != CPPMEGA_MI355_F32) {
      const uint2 r = p.y_dtype == CPPMEGA_MI355_F16 ? make_uint2(pack_f16(v[0], v[1]), pack_f16(v[2], v[3])) : make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
      __builtin_memcpy((unsigned short*)p.y + at, &r, 8);
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (n + c < p.n) store_as(p.y, at + c, p.y_dtype, v[c]);
    }
  }
}

template <int DT>
int launch(const GroupedParams& p, int tm, hipStream_t stream) {
  // every expert with rows has at least one tile of rows; at most one is not full
  const int bm = 16 * tm;
  const long long tails = p.experts + 1 < p.rows ? p.experts + 1 : p.rows;
  const long long tiles_m = p.rows / bm + tails < p.rows ? p.rows / bm + tails : p.rows;
  // Outputs of a workgroup: 64, or 16 where that leaves CUs without one (two workgroups to a CU are wanted at least)
  const bool wide = tiles_m * ((p.n + 63) / 64) >= 512;
  const long long tiles = tiles_m * ((p.n + (wide ? 63 : 15)) / (wide ? 64 : 16));
  if (tiles > 0x7fffffffll) return fail(CPPMEGA_MI355_ERR_UNSUPPORTED, "grouped_gemm: %lld tiles in one call", tiles);
  const dim3 grid((unsigned)tiles), block(64 * kWaves);
#define CM_STREAM(tm_)                                                                               \
  do {                                                                                               \
    if (wide) hipLaunchKernelGGL((grouped_stream_kernel<DT, tm_, 4>), grid, block, 0, stream, p);    \
    else hipLaunchKernelGGL((grouped_stream_kernel<DT, tm_, 1>), grid, block, 0, stream, p);         \
  } while (0)
  if (tm == 1) CM_STREAM(1);
  else if (tm == 2) CM_STREAM(2);
  else CM_STREAM(4);
#undef CM_STREAM
  CM_HIP_CHECK(hipGetLastError());
  return 0;
}

}  // namespace

int grouped_stream_launch(const GroupedParams& p, int dtype, int tm, hipStream_t stream) {
  if (dtype == CPPMEGA_MI355_E4M3) return launch<CPPMEGA_MI355_E4M3>(p, tm, stream);
  if (dtype == CPPMEGA_MI355_F16) return launch<CPPMEGA_MI355_F16>(p, tm, stream);
  return launch<CPPMEGA_MI355_BF16>(p, tm, stream);
}

}  // namespace cm

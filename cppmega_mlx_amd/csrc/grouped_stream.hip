// Products grouped by expert for few rows (gfx950): the experts' weights pass once, straight into registers.
//
// Bound by memory: an expert with 16 rows has 16 products for every weight that it reads, the matrix cores could do two hundred.  A
// workgroup has 16 rows of one expert and 64 outputs (16 where that leaves CUs without work); its four wavefronts divide the
// contraction, and their sums meet in LDS once at the end, added in order.  A step is 128 bytes of every weight row (whole cache lines),
// requested one step ahead; the activations' pieces come from the caches, a quarter of the traffic.  Which expert a workgroup has, every
// wavefront finds by itself (a scan over the counts in registers: no table, no barrier in front of the first load).
// Measured: 256 rows over 61 of 64 experts, e4m3, 4096 x 7168: 298 us = 6.0 TB/s; 8 rows of 8 experts, bf16, 4096 x 2048: 25 us = 5.3 TB/s.
// Non-temporal loads were 15 to 20 % slower, eight wavefronts 5 %, 32 or 64 rows to a workgroup 5 to 15 % at any number of rows.
//
// e4m3 codes become bfloat16 on the way, which is exact; a step is one 128-channel block, whose sum is scaled in float32.

#include <type_traits>

#include "grouped_gemm.h"

namespace cm {
namespace {

constexpr int kWaves = 4;

template <int DT, int TN>
__global__ __launch_bounds__(64 * kWaves, 2) void grouped_stream_kernel(const GroupedParams p) {
  constexpr bool FP8 = DT == CPPMEGA_MI355_E4M3, F16 = DT == CPPMEGA_MI355_F16;
  constexpr int BYTES = FP8 ? 1 : 2, STEP = 128 / BYTES, BM = 16, BN = 16 * TN;
  __shared__ f32x4 sums[kWaves][TN][64];
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
  const char* wat[TN];
  const float *sxat = nullptr, *swat = nullptr;
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int n = n0 + j * 16 + l16;
    wat[j] = (const char*)p.w + ((size_t)(e < p.experts ? e : 0) * p.n + (n < p.n ? n : p.n - 1)) * p.k * BYTES + quad * 16;
  }
  const size_t x_row = (size_t)(first + (l16 < rows ? l16 : rows - 1));      // (rows past the end repeat the last one and are not stored)
  const char* const xat = (const char*)p.x + x_row * p.x_pitch * BYTES + quad * 16;
  if (FP8) sxat = p.x_scale + x_row * (p.x_scale_block ? blocks_k : 1);
  if (FP8) swat = p.w_scale + ((size_t)(e < p.experts ? e : 0) * ((p.n + 127) / 128) + n0 / 128) * blocks_k;

  f32x4 acc[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  u32x4 w[2][TN][2], x[2][2];
  float sx[2], sw[2];
  // PART: the last step, of which a part may not be there (a condition on every load costs 15 %: its select waits for the data)
  auto load = [&](int s, int to, auto part) {
    constexpr bool PART = decltype(part)::value;
    const size_t at = (size_t)s * 128;
    const int left = p.k * BYTES - s * 128 - quad * 16;          // bytes of the row from this lane's piece on
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool there = !PART || left > 64 * h;
#pragma unroll
      for (int j = 0; j < TN; ++j) w[to][j][h] = there ? *(const u32x4*)(wat[j] + at + h * 64) : u32x4{0u, 0u, 0u, 0u};
      x[to][h] = there ? *(const u32x4*)(xat + at + h * 64) : u32x4{0u, 0u, 0u, 0u};
    }
    if (FP8) {
      sx[to] = sxat[p.x_scale_block ? s : 0];
      sw[to] = swat[s];
    }
  };
  auto multiply = [&](int b) {
    if constexpr (FP8) {
      bf16x8 xv[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) xv[c] = cvt8(x[b][c >> 1][2 * (c & 1)], x[b][c >> 1][2 * (c & 1) + 1]);
      const float f = sx[b] * sw[b];
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        f32x4 t = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < 4; ++c) t = mm<false>(cvt8(w[b][j][c >> 1][2 * (c & 1)], w[b][j][c >> 1][2 * (c & 1) + 1]), xv[c], t);
#pragma unroll
        for (int v = 0; v < 4; ++v) acc[j][v] = fmaf(f, t[v], acc[j][v]);
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[j] = mm<F16>(__builtin_bit_cast(bf16x8, w[b][j][h]), __builtin_bit_cast(bf16x8, x[b][h]), acc[j]);
    }
  };
  const std::integral_constant<bool, false> whole;
  const int end = p.k * BYTES / 128 < s1 ? p.k * BYTES / 128 : s1;
  if (s0 < end) load(s0, 0, whole);
  for (int s = s0; s < end; s += 2) {
    if (s + 1 < end) load(s + 1, 1, whole);
    multiply(0);
    if (s + 1 < end) {
      if (s + 2 < end) load(s + 2, 0, whole);
      multiply(1);
    }
  }
  if (end < s1) {
    load(end, 0, std::integral_constant<bool, true>());
    multiply(0);
  }
  // ---- the wavefronts' sums, in order; lane: row l % 16, outputs 4 (l / 16) + 0..3 of a tile ----
#pragma unroll
  for (int j = 0; j < TN; ++j) sums[wave][j][lane] = acc[j];
  __syncthreads();
  if (wave >= TN) return;
  f32x4 v = sums[0][wave][lane];
#pragma unroll
  for (int k = 1; k < kWaves; ++k) v += sums[k][wave][lane];
  const int n = n0 + wave * 16 + quad * 4;
  if (l16 >= rows || n >= p.n) return;
  const size_t at = (size_t)(first + l16) * p.y_pitch + n;
  if (n + 4 <= p.n && p.y_dtype != CPPMEGA_MI355_F32) {
    const uint2 r = p.y_dtype == CPPMEGA_MI355_F16 ? make_uint2(pack_f16(v[0], v[1]), pack_f16(v[2], v[3])) : make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
    __builtin_memcpy((unsigned short*)p.y + at, &r, 8);
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (n + c < p.n) store_as(p.y, at + c, p.y_dtype, v[c]);
  }
}

template <int DT>
int launch(const GroupedParams& p, hipStream_t stream) {
  const long long tails = p.experts + 1 < p.rows ? p.experts + 1 : p.rows;       // tiles of rows that are not full, at most
  const long long tiles_m = p.rows / 16 + tails < p.rows ? p.rows / 16 + tails : p.rows;
  const bool wide = tiles_m * ((p.n + 63) / 64) >= 512;                          // (two workgroups to a CU at least)
  const long long tiles = tiles_m * (wide ? (p.n + 63) / 64 : (p.n + 15) / 16);
  if (int rc = check_tiles(tiles, 64 * kWaves)) return rc;
  const dim3 grid((unsigned)tiles), block(64 * kWaves);
  if (wide) hipLaunchKernelGGL((grouped_stream_kernel<DT, 4>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((grouped_stream_kernel<DT, 1>), grid, block, 0, stream, p);
  CM_HIP_CHECK(hipGetLastError());
  return 0;
}

}  // namespace

int grouped_stream_launch(const GroupedParams& p, int dtype, hipStream_t stream) {
  if (dtype == CPPMEGA_MI355_E4M3) return launch<CPPMEGA_MI355_E4M3>(p, stream);
  if (dtype == CPPMEGA_MI355_F16) return launch<CPPMEGA_MI355_F16>(p, stream);
  return launch<CPPMEGA_MI355_BF16>(p, stream);
}

}  // namespace cm

// Products with 4-bit weights and group scales for few rows, dense or by expert, plain or gated (gfx950).
//
//   y[t, n] = sum_k x[t, k] (s[n, g] q[n, k] + b[n, g]),  g = k / G;  without biases b = -8 s
//
// Bound by memory: the weights pass once.  A workgroup has 16 TM rows of one expert and 16 TN rows of its weight (gated: half of them
// the gate's); its wavefronts divide the contraction, and their sums meet in LDS once at the end, added in order.
// Four bits become 16 + q in 16 bits by a shift and an and-or, two at a time: q lies where float16 and bfloat16 between 16 and 32 have their
// next four bits.  Products are exact; 16 times a group's sum of x comes off again in float32 with the bias,
//   sum over a group = s (sum x (16 + q)) + (b - 16 s) (sum x),
// where sum x comes from the matrix cores too (times ones), once for all of a workgroup's weights.
// x is the first operand: a lane has one row of the weight in every sum, and with it one scale and one bias.
// A step is 128 channels, 16 bytes (32 codes) a lane; a word of it is eight channels, of which the low and the high half of a register
// take those four apart, so the pieces of x are put in that order.  With groups below 128 the four words of the four lanes of a row change
// places, so that one instruction has 32 channels in a run.

#include <string.h>

#include <type_traits>

#include "grouped_gemm.h"

namespace cm {
namespace {

constexpr int kMostWaves = 8;

struct W4Params {
  GroupedParams g;                                               // (w, scales: of 2 n rows when gated)
  const void *scale, *bias;
  int gated;
};

// Eight codes as 16 + q in 16 bits, in the order 0 4 1 5 2 6 3 7.
template <bool F16>
__device__ __forceinline__ bf16x8 widen(unsigned w) {
  constexpr unsigned mask = F16 ? 0x03c003c0u : 0x00780078u, one = F16 ? 0x4c004c00u : 0x41804180u;
  u32x4 r;
  if (F16) r = u32x4{w << 6, w << 2, w >> 2, w >> 6};
  else r = u32x4{w << 3, w >> 1, w >> 5, w >> 9};
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = (r[i] & mask) | one;
  return __builtin_bit_cast(bf16x8, r);
}
// Eight values of x in the same order.
__device__ __forceinline__ bf16x8 reorder(const u32x4 x) {
  return __builtin_bit_cast(bf16x8, u32x4{__builtin_amdgcn_perm(x[2], x[0], 0x05040100u), __builtin_amdgcn_perm(x[2], x[0], 0x07060302u),
                                          __builtin_amdgcn_perm(x[3], x[1], 0x05040100u), __builtin_amdgcn_perm(x[3], x[1], 0x07060302u)});
}
// Words of four quads of lanes: word i of quad j becomes word j of quad i.
__device__ __forceinline__ void transpose4(u32x4& w) {
  u32x2 a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false), b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
  const u32x2 c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false), d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  w = u32x4{c[0], c[1], d[0], d[1]};
}

// The scales (or biases) of N consecutive groups as they are stored, S bytes each.
template <int N, int S>
struct Groups {
  unsigned v[(N * S + 3) / 4];
  __device__ __forceinline__ void load(const void* base, size_t at) { __builtin_memcpy(v, (const char*)base + at * S, N * S); }
  __device__ __forceinline__ void load_part(const void* base, size_t at, int left) {       // zeros for groups that are not there
#pragma unroll
    for (int i = 0; i < (N * S + 3) / 4; ++i) v[i] = 0u;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i >= left) continue;
      if (S == 4) v[i] = ((const unsigned*)base)[at + i];
      else v[i / 2] |= (unsigned)((const unsigned short*)base)[at + i] << (16 * (i & 1));
    }
  }
  template <bool F16>
  __device__ __forceinline__ float get(int i) const {
    if (S == 4) return __uint_as_float(v[i]);
    const unsigned short b = (unsigned short)(v[i / 2] >> (16 * (i & 1)));
    return F16 ? f16_bits_to_f32(b) : bf16_bits_to_f32(b);
  }
};

// S: bytes of a scale.
template <int G, int TN, int TM, bool F16, int S>
__global__ __launch_bounds__(64 * kMostWaves, 2) void w4_kernel(const W4Params p) {
  constexpr int kSteps = TM == 1 && G > 32 ? 2 : 1;                        // (two rounds of operands are in registers)
  constexpr int kRound = 128 * kSteps, kGroups = kRound / G;     // channels and groups of a round
  constexpr int kIn = G / 32;                                    // matrix instructions to a group
  constexpr bool SWAP = G < 128;
  extern __shared__ f32x4 sums[];                                // [wavefronts][TM][TN][64]
  const GroupedParams& q = p.g;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), waves = (int)blockDim.x >> 6;
  const int l16 = lane & 15, quad = lane >> 4;
  const int to = p.gated ? TN / 2 : TN;                          // outputs of a workgroup, in 16s
  const int tiles_n = (q.n + 16 * to - 1) / (16 * to);
  const int mt = (int)(blockIdx.x / (unsigned)tiles_n), n0 = (int)(blockIdx.x % (unsigned)tiles_n) * 16 * to;
  int e, first, rows;
  if (!rows_of_tile<16 * TM>(q, mt, e, first, rows)) return;
  const int expert = e < q.experts ? e : 0;
  const int groups = q.k / G;
  const int rounds = e < q.experts ? (q.k + kRound - 1) / kRound : 0, whole = q.k / kRound;
  const int r0 = (int)((long long)rounds * wave / waves), r1 = (int)((long long)rounds * (wave + 1) / waves);

  const char* wat[TN];
  size_t sat[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int up = j >= to ? 1 : 0, n = n0 + (j - (up ? to : 0)) * 16 + l16;
    const size_t row = (size_t)expert * (p.gated ? 2 : 1) * q.n + (n < q.n ? n : q.n - 1) + (up ? q.n : 0);
    wat[j] = (const char*)q.w + row * (q.k >> 1) + quad * 16;
    sat[j] = row * groups;
  }
  const char* xat[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int row = i * 16 + l16;                                // (rows past the end repeat the last one and are not stored)
    xat[i] = (const char*)q.x + ((size_t)(first + (row < rows ? row : rows - 1)) * q.x_pitch + quad * (SWAP ? 8 : 32)) * 2;
  }

  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  u32x4 w[2][TN][kSteps], x[2][TM][4 * kSteps];
  Groups<kGroups, S> s[2][TN], b[2][TN];
  // Round r into buffer `at`.  PART: the last one, of which a part may not be there: zeros for x, of which nothing is added.
  auto load = [&](int r, int at, auto part) __attribute__((always_inline)) {
    constexpr bool PART = decltype(part)::value;
    const int left = q.k - r * kRound;                           // channels from this round on
#pragma unroll
    for (int j = 0; j < TN; ++j) {
#pragma unroll
      for (int h = 0; h < kSteps; ++h) {
        if (!PART || h * 128 + quad * 32 < left) __builtin_memcpy(&w[at][j][h], wat[j] + (size_t)r * (kRound / 2) + h * 64, 16);
        else w[at][j][h] = u32x4{0u, 0u, 0u, 0u};
      }
      const size_t group = sat[j] + (size_t)r * kGroups;
      if (PART) s[at][j].load_part(p.scale, group, left / G);
      else s[at][j].load(p.scale, group);
      if (p.bias) {
        if (PART) b[at][j].load_part(p.bias, group, left / G);
        else b[at][j].load(p.bias, group);
      }
    }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int c = 0; c < 4 * kSteps; ++c) {
        // channels of this lane's piece: of 32 in a run (SWAP), or of its 32 of a step
        const int in = (c >> 2) * 128 + (SWAP ? (c & 3) * 32 : (c & 3) * 8), first_k = in + quad * (SWAP ? 8 : 32);
        if (!PART || first_k < left) __builtin_memcpy(&x[at][i][c], xat[i] + ((size_t)r * kRound + in) * 2, 16);
        else x[at][i][c] = u32x4{0u, 0u, 0u, 0u};
      }
  };
  const bf16x8 ones = __builtin_bit_cast(bf16x8, F16 ? u32x4{0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u} : u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});
  auto multiply = [&](int at) __attribute__((always_inline)) {
    if (SWAP)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int h = 0; h < kSteps; ++h) transpose4(w[at][j][h]);
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      f32x4 t[TM][TN], sum[TM];
#pragma unroll
      for (int c = g * kIn; c < (g + 1) * kIn; ++c) {
        bf16x8 xv[TM];
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          xv[i] = reorder(x[at][i][c]);
          sum[i] = mm<F16>(xv[i], ones, c == g * kIn ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : sum[i]);
        }
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const bf16x8 wv = widen<F16>(w[at][j][c >> 2][c & 3]);
#pragma unroll
          for (int i = 0; i < TM; ++i) t[i][j] = mm<F16>(xv[i], wv, c == g * kIn ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : t[i][j]);
        }
      }
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const float f = s[at][j].template get<F16>(g), off = p.bias ? fmaf(-16.0f, f, b[at][j].template get<F16>(g)) : -24.0f * f;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int v = 0; v < 4; ++v) acc[i][j][v] = fmaf(f, t[i][j][v], fmaf(off, sum[i][v], acc[i][j][v]));
      }
    }
  };
  const std::integral_constant<bool, false> all;
  const int end = whole < r1 ? whole : r1;
  if (r0 < end) load(r0, 0, all);
  for (int r = r0; r < end; r += 2) {
    if (r + 1 < end) load(r + 1, 1, all);
    multiply(0);
    if (r + 1 < end) {
      if (r + 2 < end) load(r + 2, 0, all);
      multiply(1);
    }
  }
  if (r0 <= whole && whole < r1) {
    load(whole, 0, std::integral_constant<bool, true>());
    multiply(0);
  }

  // ---- the wavefronts' sums, in order; lane: weight row l % 16, rows 4 (l / 16) + 0..3 of a tile ----
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) sums[((wave * TM + i) * TN + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  auto sum_of = [&](int i, int j) {
    f32x4 v = sums[(i * TN + j) * 64 + lane];
    for (int k = 1; k < waves; ++k) v += sums[((k * TM + i) * TN + j) * 64 + lane];
    return v;
  };
  for (int u = wave; u < TM * to; u += waves) {
    const int i = u / to, j = u - i * to, n = n0 + j * 16 + l16;
    f32x4 v = sum_of(i, j);
    if (p.gated) {
      const f32x4 up = sum_of(i, to + j);
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = gated(v[c], up[c], q.activation);
    }
    if (n >= q.n) continue;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int row = i * 16 + quad * 4 + c;
      if (row < rows) store_as(q.y, (size_t)(first + row) * q.y_pitch + n, q.y_dtype, v[c]);
    }
  }
}

template <int G, bool F16, int S>
int launch(const W4Params& p, hipStream_t stream) {
  const GroupedParams& q = p.g;
  // rows to a workgroup: as many as an expert has on average, up to 32
  const long long mean = (q.rows + q.experts - 1) / q.experts;
  const int tm = mean <= 16 ? 1 : 2;
  const long long bm = 16 * tm, tails = q.experts + 1 < q.rows ? q.experts + 1 : q.rows;
  const long long tiles_m = !q.offsets ? (q.rows + bm - 1) / bm : q.rows / bm + tails < q.rows ? q.rows / bm + tails : q.rows;
  auto tiles = [&](int tn) { return tiles_m * ((q.n + 16 * tn / (p.gated ? 2 : 1) - 1) / (16 * tn / (p.gated ? 2 : 1))); };
  const int least = p.gated || tm > 1 ? 2 : 1;
  const int tn = least < 2 && tiles(2) < 512 ? 1 : 2;
  const long long count = tiles(tn);
  const int rounds = tm == 1 && G > 32 ? (q.k + 255) / 256 : (q.k + 127) / 128;
  int waves = 4;
  while (waves < kMostWaves && waves < rounds && count * waves < 2048) waves *= 2;
  if (int rc = check_tiles(count, 64 * waves)) return rc;
  const dim3 grid((unsigned)count), block(64 * waves);
  const size_t lds = (size_t)waves * tm * tn * 64 * sizeof(f32x4);
#define CM_W4(tn_, tm_) hipLaunchKernelGGL((w4_kernel<G, tn_, tm_, F16, S>), grid, block, lds, stream, p)
  if (tm == 2) CM_W4(2, 2);
  else if (tn == 2) CM_W4(2, 1);
  else CM_W4(1, 1);
#undef CM_W4
  CM_HIP_CHECK(hipGetLastError());
  return 0;
}

template <int G>
int launch_group(const W4Params& p, bool f16, bool wide, hipStream_t stream) {
  if (wide) return f16 ? launch<G, true, 4>(p, stream) : launch<G, false, 4>(p, stream);
  return f16 ? launch<G, true, 2>(p, stream) : launch<G, false, 2>(p, stream);
}

}  // namespace

int w4_gemm_launch(const cppmega_mi355_w4_gemm_args_t& a, hipStream_t stream) {
  const bool is_gated = a.activation != CPPMEGA_MI355_GATE_NONE;
  if (is_gated && a.activation != CPPMEGA_MI355_GATE_SILU && a.activation != CPPMEGA_MI355_GATE_GELU_TANH)
    return fail(CPPMEGA_MI355_ERR_SHAPE, "w4_gemm: unknown activation %d", a.activation);
  if (a.rows < 0 || a.rows > 0x1fffffffll || a.experts < 1 || a.n < 1 || a.k < 1)
    return fail(CPPMEGA_MI355_ERR_SHAPE, "w4_gemm: rows=%lld experts=%d n=%d k=%d", (long long)a.rows, a.experts, a.n, a.k);
  if (a.n > (is_gated ? CPPMEGA_MI355_GATED_MAX_OUTPUTS : CPPMEGA_MI355_GROUPED_MAX_SIZE) || a.k > CPPMEGA_MI355_GROUPED_MAX_SIZE)
    return fail(CPPMEGA_MI355_ERR_SHAPE, "w4_gemm: n=%d k=%d, at most 2^30 weight rows and channels are served", a.n, a.k);
  if (a.experts > kMaxExperts) return fail(CPPMEGA_MI355_ERR_UNSUPPORTED, "w4_gemm: %d experts, at most %d are served", a.experts, kMaxExperts);
  if (a.group != 32 && a.group != 64 && a.group != 128) return fail(CPPMEGA_MI355_ERR_SHAPE, "w4_gemm: groups of %d, 32, 64 and 128 are served", a.group);
  if (a.k % a.group != 0) return fail(CPPMEGA_MI355_ERR_SHAPE, "w4_gemm: k=%d is no multiple of the group, %d", a.k, a.group);
  if (a.x_dtype != CPPMEGA_MI355_F16 && a.x_dtype != CPPMEGA_MI355_BF16)
    return fail(CPPMEGA_MI355_ERR_DTYPE, "w4_gemm: rows of dtype %d are not float16 / bfloat16", a.x_dtype);
  if (a.y_dtype != CPPMEGA_MI355_F32 && a.y_dtype != a.x_dtype) return fail(CPPMEGA_MI355_ERR_DTYPE, "w4_gemm: a result of dtype %d from rows of dtype %d", a.y_dtype, a.x_dtype);
  if (a.scale_dtype != CPPMEGA_MI355_F32 && a.scale_dtype != a.x_dtype)
    return fail(CPPMEGA_MI355_ERR_DTYPE, "w4_gemm: scales of dtype %d beside rows of dtype %d", a.scale_dtype, a.x_dtype);
  if (a.offsets_dtype != CPPMEGA_MI355_I32 && a.offsets_dtype != CPPMEGA_MI355_I64) return fail(CPPMEGA_MI355_ERR_DTYPE, "w4_gemm: offsets must be int32 or int64");
  if (a.rows == 0) return 0;
  if (!a.x || !a.w || !a.scale || !a.y || (!a.offsets && a.experts != 1)) return fail(CPPMEGA_MI355_ERR_NULL, "w4_gemm: x / w / scale / y / offsets is NULL");
  W4Params p;
  memset(&p, 0, sizeof(p));
  GroupedParams& q = p.g;
  q.x = a.x; q.w = a.w; q.y = a.y; q.offsets = a.offsets;
  q.rows = a.rows; q.x_pitch = a.x_pitch; q.y_pitch = a.y_pitch;
  q.experts = a.experts; q.n = a.n; q.k = a.k;
  q.y_dtype = a.y_dtype; q.offsets64 = a.offsets_dtype == CPPMEGA_MI355_I64; q.zero_tail = a.zero_tail; q.activation = a.activation;
  p.scale = a.scale; p.bias = a.bias; p.gated = is_gated;
  const bool f16 = a.x_dtype == CPPMEGA_MI355_F16, wide = a.scale_dtype == CPPMEGA_MI355_F32;
  return a.group == 32 ? launch_group<32>(p, f16, wide, stream) : a.group == 64 ? launch_group<64>(p, f16, wide, stream) : launch_group<128>(p, f16, wide, stream);
}

}  // namespace cm

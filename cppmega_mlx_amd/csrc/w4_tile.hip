// Products with 4-bit weights and group scales for many rows of an expert: a weight is widened once for 64 rows (gfx950).
//
// A workgroup has 64 rows of x of one expert and SLICES ways to divide the contraction: its other wavefronts are pairs of 16 rows of the weight
// (gated: the same 16 outputs of the gate and of the up projection).  A pass is 1024 channels: x comes through registers into LDS in the codes'
// order while the pass before is multiplied, and every slice takes 8 / SLICES steps of it, whose codes were asked for a pass ahead.
// The sums of x over a group are the matrix cores' too, each once in the workgroup, and go through LDS.  Channels that are not there are
// zeros of x, and their scales count as zero.
//
// Bound by the matrix cores, the vector instructions that widen and scale, and reads of x from LDS, a third of the time each, which the
// two wavefronts of a SIMD overlap little (a set order of instructions changed nothing); a pass takes 4 us and more, the memory's answer to the
// requests made a pass ahead.  Bfloat16, groups of 128: 512 x 8192 x 8192 109 us, 0.63 PFLOP/s; 4096 x 4096 x 4096 242 us, 0.57; groups of 64, which
// change places and are scaled twice as often: 135 and 303.

#include "w4.h"

namespace cm {
namespace {

constexpr int kRowTiles = 4, kBM = 16 * kRowTiles, kSteps = 8, kWaves = 8, kPieces = 16;   // steps of a pass; pieces of x of a thread
constexpr int kX = kBM * kSteps * 16;                            // u32x4s of x

template <int G, bool F16, int S, int SLICES>
__global__ __launch_bounds__(64 * kWaves, 2) void w4_tile_kernel(const W4Params p) {
  constexpr int kIn = G / 32, kPer = 4 / kIn;                    // 32s of channels in a group, groups in a step
  constexpr int kMine = kSteps / SLICES, kPairs = kWaves / SLICES, kSums = kRowTiles / kPairs;   // row tiles whose sums of x a wavefront makes
  constexpr bool SWAP = G < 128;
  __shared__ u32x4 smem[kX];                                     // x, afterwards the slices' sums
  __shared__ float xsum[kSteps][kPer][kBM];                      // of a pass
  static_assert(kMine <= 4 && kPairs <= kRowTiles, "a quad of lanes has the groups of one step, a pair one row tile's sums or more");
  static_assert(kX >= kWaves * 2 * kRowTiles * 64, "the slices' sums lie where x was");
  const GroupedParams& q = p.g;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int l16 = lane & 15, quad = lane >> 4, slice = wave % SLICES, pair = wave / SLICES;
  const int mt = p.tile0 + (int)blockIdx.y;
  int e = 0, first = mt * kBM, rows = (int)(q.rows - first);
  if (q.offsets && !rows_of_tile<kBM>(q, mt, e, first, rows)) return;
  e = __builtin_amdgcn_readfirstlane(e);
  first = __builtin_amdgcn_readfirstlane(first);
  rows = __builtin_amdgcn_readfirstlane(rows < kBM ? rows : kBM);
  const bool there = e < q.experts;
  const int groups = q.k / G, pitch = q.k >> 1, steps = there ? (q.k + 127) / 128 : 0;

  // ---- a pair's weights: their places, and 32 bits of the lane ----
  const int across = (p.gated ? 16 : 32) * kPairs, n0 = (int)blockIdx.x * across + pair * (p.gated ? 16 : 32);
  const char *wt[2], *st[2], *bt[2];
  unsigned wo[2], go[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int n = n0 + (p.gated ? 0 : 16 * j), n1 = n < q.n ? n : q.n - 1, row = n + l16 < q.n ? l16 : q.n - 1 - n1;
    const size_t weight = (size_t)(there ? e : 0) * (p.gated ? 2 : 1) * q.n + (p.gated && j ? q.n : 0) + n1;
    wt[j] = (const char*)q.w + weight * pitch;
    st[j] = (const char*)p.scale + weight * groups * S;
    bt[j] = (const char*)p.bias + weight * groups * S;
    wo[j] = (unsigned)row * (unsigned)pitch;
    go[j] = (unsigned)row * (unsigned)groups * S;
  }
  u32x4 w[2][kMine];
  // (codes behind the row's end: its last ones, whose x is zero)
  auto load_w = [&](int j, int i, int base) __attribute__((always_inline)) {
    const int at = (base + slice * kMine + i) * 64 + quad * 16;
    __builtin_memcpy(&w[j][i], wt[j] + wo[j] + (unsigned)(at < pitch - 16 ? at : pitch - 16), 16);
  };
  // Quad i has the groups of the slice's step i; zeros for those that are not there.
  struct Factors {
    float scale[kPer], off[kPer];
  };
  Factors now[2];
  unsigned raw_scale[2][kPer], raw_bias[2][kPer];
  const float shift = p.bias ? -16.0f : -24.0f;
  auto load_groups = [&](int base) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int g = 0; g < kPer; ++g) {
        const int group = (base + slice * kMine + quad) * kPer + g;
        const unsigned at = go[j] + (unsigned)(group < groups ? group : groups - 1) * S;
        if (S == 4) raw_scale[j][g] = *(const unsigned*)(st[j] + at);
        else raw_scale[j][g] = *(const unsigned short*)(st[j] + at);
        if (!p.bias) raw_bias[j][g] = 0u;
        else if (S == 4) raw_bias[j][g] = *(const unsigned*)(bt[j] + at);
        else raw_bias[j][g] = *(const unsigned short*)(bt[j] + at);
      }
  };
  auto value = [](unsigned v) { return S == 4 ? __uint_as_float(v) : F16 ? f16_bits_to_f32((unsigned short)v) : bf16_bits_to_f32((unsigned short)v); };
  auto take_groups = [&](int base) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int g = 0; g < kPer; ++g) {
        const bool mine = quad < kMine && (base + slice * kMine + quad) * kPer + g < groups;
        const float s = value(raw_scale[j][g]);
        now[j].scale[g] = mine ? s : 0.0f;
        now[j].off[g] = mine ? fmaf(shift, s, value(raw_bias[j][g])) : 0.0f;
      }
  };

  // ---- x: a thread has one piece (eight channels) of every fourth row ----
  const char* const xb = (const char*)q.x + (size_t)first * q.x_pitch * 2;
  const int piece = (int)threadIdx.x & 127, xrow = (int)threadIdx.x >> 7;
  u32x4 v[kPieces];
  auto fetch = [&](int base) __attribute__((always_inline)) {
    int channel = base * 128 + piece * 8;
    channel = channel < q.k ? channel : 0;
    int row = xrow;
    asm("" : "+v"(row));                                         // (the places are made here, not kept in registers throughout)
#pragma unroll
    for (int u = 0; u < kPieces; ++u) {
      const int r = row + 4 * u < rows ? row + 4 * u : rows - 1;
      __builtin_memcpy(&v[u], xb + ((unsigned)r * (unsigned)q.x_pitch + (unsigned)channel) * 2u, 16);
    }
  };
  auto put = [&](int base) __attribute__((always_inline)) {
    const bool here = base * 128 + piece * 8 < q.k;
#pragma unroll
    for (int u = 0; u < kPieces; ++u) {
      const u32x4 x = here ? v[u] : u32x4{0u, 0u, 0u, 0u};
      smem[piece * kBM + ((xrow + 4 * u) ^ (piece & 15))] = __builtin_bit_cast(u32x4, reorder(x));
    }
  };
  // (piece o of row r lies at 64 o + (r ^ (o % 16)): 16 pieces of a row and 16 rows of a piece begin in different banks)
  const u32x4* at_x[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int o = SWAP ? c * 4 + quad : quad * 4 + c;
    at_x[c] = smem + (size_t)slice * kMine * 16 * kBM + o * kBM + (l16 ^ o);
  }

  const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
  f32x4 acc[2][kRowTiles];
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int i = 0; i < kRowTiles; ++i) acc[j][i] = zero;
  unsigned sixteen = F16 ? 0x4c004c00u : 0x41804180u;
  asm("" : "+v"(sixteen));
  const bf16x8 ones = __builtin_bit_cast(bf16x8, F16 ? u32x4{0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u} : u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});
  if (steps > 0) {
    fetch(0);
    load_groups(0);
#pragma unroll
    for (int i = 0; i < kMine; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) load_w(j, i, 0);
  }
  for (int base = 0; base < steps; base += kSteps) {
    put(base);
    __syncthreads();
    take_groups(base);
    // (behind the last pass the rows' ends again: no branch, across which the compiler would move products)
    fetch(base + kSteps);
    load_groups(base + kSteps);
    __builtin_amdgcn_sched_barrier(0);
    each<kMine>([&](auto step) __attribute__((always_inline)) {
      constexpr int I = decltype(step)::value;
      if (SWAP) {
        transpose4(w[0][I]);
        transpose4(w[1][I]);
      }
      f32x4 t[2][kRowTiles], one[kSums];
      each<4>([&](auto c_) __attribute__((always_inline)) {
        constexpr int c = decltype(c_)::value, g = c / kIn;
        constexpr bool fresh = c % kIn == 0;
        bf16x8 xv[kRowTiles];
#pragma unroll
        for (int i = 0; i < kRowTiles; ++i) xv[i] = __builtin_bit_cast(bf16x8, at_x[c][I * 16 * kBM + i * 16]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const bf16x8 codes = widen<F16>(w[j][I][c], sixteen);
#pragma unroll
          for (int i = 0; i < kRowTiles; ++i) t[j][i] = mm<F16>(xv[i], codes, fresh ? zero : t[j][i]);
        }
        // this wavefront's share of the sums of x (read again: no branch here, across which the compiler would move products)
#pragma unroll
        for (int i = 0; i < kSums; ++i)
          one[i] = mm<F16>(ones, __builtin_bit_cast(bf16x8, at_x[c][I * 16 * kBM + (pair * kSums + i) * 16]), fresh ? zero : one[i]);
        if constexpr (c % kIn == kIn - 1) {
#pragma unroll
          for (int i = 0; i < kSums; ++i) xsum[slice * kMine + I][g][(pair * kSums + i) * 16 + l16] = one[i][0];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float f = __uint_as_float(of_quad<I>(__float_as_uint(now[j].scale[g])));
#pragma unroll
            for (int i = 0; i < kRowTiles; ++i)
#pragma unroll
              for (int r = 0; r < 4; ++r) acc[j][i][r] = fmaf(f, t[j][i][r], acc[j][i][r]);
          }
        }
      });
      load_w(0, I, base + kSteps);
      load_w(1, I, base + kSteps);
      __builtin_amdgcn_sched_barrier(0);
    });
    __syncthreads();
    // the part that goes by the sums of x: four steps of a slice (or as many as it has) to an instruction
#pragma unroll
    for (int g = 0; g < kPer; ++g)
#pragma unroll
      for (int i = 0; i < kRowTiles; ++i) {
        const float x = xsum[slice * kMine + (quad & (kMine - 1))][g][i * 16 + l16];    // (quads without a step have factors of zero)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(x, now[j].off[g], acc[j][i], 0, 0, 0);
      }
  }

  // ---- the slices' sums, in order; lane: weight row l % 16, rows 4 (l / 16) + 0..3 of a row tile ----
  f32x4* const sums = reinterpret_cast<f32x4*>(smem);            // [pairs][row tiles][2][slices][64]
#pragma unroll
  for (int i = 0; i < kRowTiles; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) sums[(((pair * kRowTiles + i) * 2 + j) * SLICES + slice) * 64 + lane] = acc[j][i];
  __syncthreads();
  for (int u = wave; u < kPairs * kRowTiles; u += kWaves) {
    f32x4 y[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      y[j] = sums[(u * 2 + j) * SLICES * 64 + lane];
#pragma unroll
      for (int s = 1; s < SLICES; ++s) y[j] += sums[((u * 2 + j) * SLICES + s) * 64 + lane];
    }
    const int row = u % kRowTiles * 16 + quad * 4, n = (int)blockIdx.x * across + u / kRowTiles * (p.gated ? 16 : 32) + l16;
    auto store = [&](int at, int r, float value) {
      if (at < q.n && row + r < rows) store_as(q.y, (size_t)(first + row + r) * q.y_pitch + at, q.y_dtype, value);
    };
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (p.gated) {
        store(n, r, gated(y[0][r], y[1][r], q.activation));
      } else {
        store(n, r, y[0][r]);
        store(n + 16, r, y[1][r]);
      }
    }
  }
}

template <int G, bool F16, int S, int SLICES>
int launch(W4Params p, hipStream_t stream) {
  const GroupedParams& q = p.g;
  const long long tails = q.experts + 1 < q.rows ? q.experts + 1 : q.rows;        // tiles of rows that are not full, at most
  const long long tiles_m = !q.offsets ? (q.rows + kBM - 1) / kBM : q.rows / kBM + tails;
  const int out = (p.gated ? 16 : 32) * (kWaves / SLICES), parts = (q.n + out - 1) / out;
  if (int rc = check_tiles("w4_gemm", parts, 64 * kWaves)) return rc;
  constexpr long long kMostY = 65535;                            // (of a grid)
  for (long long t = 0; t < tiles_m; t += kMostY) {
    p.tile0 = (int)t;
    const dim3 grid((unsigned)parts, (unsigned)(tiles_m - t < kMostY ? tiles_m - t : kMostY));
    hipLaunchKernelGGL((w4_tile_kernel<G, F16, S, SLICES>), grid, dim3(64 * kWaves), 0, stream, p);
  }
  CM_HIP_CHECK(hipGetLastError());
  return 0;
}

template <int G, bool F16, int S>
int choose(const W4Params& p, hipStream_t stream) {
  const GroupedParams& q = p.g;
  // Four slices while that leaves one workgroup to a CU.  Measured, us 2 / 4 slices, rows x n x k, bfloat16, groups of 64, biases, weights from memory: 200 x
  // 4096 x 4096 38 / 28, 48 x 16384 x 8192 67 / 52, 64 x 8192 x 8192 69 / 54, 64 x 32768 x 1024 18 / 24, 512 x 8192 x 8192 136 / 204; where the rule takes the slower
  // one: 300 x 8 experts x 2048 x 4096 39 / 31.
  const long long work = ((q.rows + kBM - 1) / kBM + q.experts / 2) * (((long long)q.n * (p.gated ? 2 : 1) + 31) / 32);   // pairs, for 64 rows each
  return work <= 512 ? launch<G, F16, S, 4>(p, stream) : launch<G, F16, S, 2>(p, stream);
}

template <int G>
int of_group(const W4Params& p, bool f16, bool wide, hipStream_t stream) {
  if (wide) return f16 ? choose<G, true, 4>(p, stream) : choose<G, false, 4>(p, stream);
  return f16 ? choose<G, true, 2>(p, stream) : choose<G, false, 2>(p, stream);
}

}  // namespace

int w4_tile_launch(const W4Params& p, int group, bool f16, bool wide, hipStream_t stream) {
  return group == 32 ? of_group<32>(p, f16, wide, stream) : group == 64 ? of_group<64>(p, f16, wide, stream) : of_group<128>(p, f16, wide, stream);
}

}  // namespace cm

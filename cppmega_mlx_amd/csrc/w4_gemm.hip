// Products with 4-bit weights and group scales for few rows, dense or by expert, plain or gated (gfx950).
//
//   y[t, n] = sum_k x[t, k] (s[n, g] q[n, k] + b[n, g]),  g = k / G;  without biases b = -8 s
//
// Widened once for 16 rows of x.  A workgroup has 16 rows of x of one expert and up to four tiles of 16 rows of its weight (gated: as many of the
// gate's as of the up projection's), a tile to a wavefront; the others divide the contraction, and their sums meet in LDS once at the
// end, added in order.  A wavefront has 8 KiB of weights on their way and nothing else: loads return in the order in which they were asked for, and
// rows of x, from the cache but behind weights, waited for memory.  x passes through LDS instead, as much of it at a time as there is room,
// in the codes' order.
//
// Times in this file: bfloat16, groups of 64, biases, and weights that come from memory (1.2 GB of them in turn), unless it says otherwise.
// Many experts are bound by memory: 61 experts of 4096 x 7168 codes in 244 us.  They read 1378 MiB (counted) where codes, scales and
// biases are 961, which fits lines of scales that come anew for every eight steps, 32 bytes of a row.  One matrix leaves a
// CU one or two workgroups, whose wavefronts wait for half of their time (16 x 16384 x 7168, float16, groups of 128: waits 0.52 of the wavefronts' cycles, vector
// instructions 0.26 and matrix ones 0.11 of the SIMDs'): for the start (arguments, x into LDS, the first weights: 4 to 5 us), for memory, and at
// the end for each other's sums.  16 x 16384 x 7168 27.5 us (float16, groups of 128, no biases 25, and 21 where the weights are in the last-level
// cache); 1 x 2048 x 7168 9.5.  Tried at 1 x 16384 x 7168 (float16, groups of 128, no biases: 19) with nothing gained, 18 to 21 us: two or four tiles to
// a wavefront, x kept in registers, 16 steps of weights on their way, 16 wavefronts, x read past LDS (as much of the first-level cache's time as the weights).

#include <string.h>

#include "w4.h"

namespace cm {
namespace {

constexpr int kMostWaves = 8, kRoom = 8192;                      // wavefronts of a workgroup; bytes of LDS that each of them brings for x

// The scales (or biases) of N consecutive groups as they are stored, S bytes each.
template <int N, int S>
struct Groups {
  static constexpr int kWords = (N * S + 3) / 4;
  unsigned v[kWords];
  __device__ __forceinline__ void load(const char* at) { __builtin_memcpy(v, at, N * S); }
  __device__ __forceinline__ void load_part(const char* at, int left) {         // zeros for groups that are not there
#pragma unroll
    for (int i = 0; i < kWords; ++i) v[i] = 0u;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i >= left) continue;
      if (S == 4) v[i] = *(const unsigned*)(at + 4 * i);
      else v[i / 2] |= (unsigned)*(const unsigned short*)(at + 2 * i) << (16 * (i & 1));
    }
  }
  // the second half in the first one's place
  __device__ __forceinline__ void drop_half(bool yes) {
    constexpr int kHalf = N * S / 8;
    if constexpr (kHalf == 0) v[0] = yes ? v[0] >> 16 : v[0];
#pragma unroll
    for (int i = 0; i < kHalf; ++i) v[i] = yes ? v[i + kHalf] : v[i];
  }
  template <bool F16>
  static __device__ __forceinline__ float value(unsigned word, int i) {
    if (S == 4) return __uint_as_float(word);
    const unsigned short b = (unsigned short)(word >> (16 * (i & 1)));
    return F16 ? f16_bits_to_f32(b) : bf16_bits_to_f32(b);
  }
};

// S: bytes of a scale.
template <int G, bool F16, int S>
__global__ __launch_bounds__(64 * kMostWaves, 4) void w4_kernel(const W4Params p) {
  constexpr int kIn = G / 32, kPer = 4 / kIn;                    // 32s of channels in a group, groups in a step
  constexpr bool SWAP = G < 128;
  extern __shared__ u32x4 smem[];                                // x, afterwards the sums
  const GroupedParams& q = p.g;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), waves = (int)blockDim.x >> 6;
  const int l16 = lane & 15, quad = lane >> 4;
  const int split = 1 << p.log_split, tiles = waves >> p.log_split, tile = wave >> p.log_split, slice = wave & (split - 1);
  const int to = p.gated ? tiles >> 1 : tiles;                   // outputs of a workgroup, in 16s
  const int up = tile >= to ? 1 : 0, n0 = ((int)blockIdx.x * to + tile - up * to) * 16;
  const int mt = p.tile0 + (int)blockIdx.y;
  int e = 0, first = mt * 16, rows = (int)(q.rows - first);
  if (q.offsets && !rows_of_tile<16>(q, mt, e, first, rows)) return;
  e = __builtin_amdgcn_readfirstlane(e);
  first = __builtin_amdgcn_readfirstlane(first);
  rows = __builtin_amdgcn_readfirstlane(rows < 16 ? rows : 16);
  const bool there = e < q.experts;
  const int groups = q.k / G, pitch = q.k >> 1, steps = there ? q.k / 128 : 0;

  // ---- passes of x through LDS: rows of it, as a power of two, and steps of a wavefront (whole blocks of eight where there is room) ----
  const int log_rows = rows > 1 ? 32 - __builtin_clz(rows - 1) : 0, row_mask = (1 << log_rows) - 1;
  const int room = waves * kRoom >> (log_rows + 8 + p.log_split), most = room >= 8 ? room & ~7 : room;
  const int per_pass = most << p.log_split;
  const char* const xb = (const char*)q.x + (size_t)first * q.x_pitch * 2;
  // piece o (eight channels) of row r of a pass: a row's pieces lie in different banks, and so do the rows' of one piece
  auto place = [&](int o, int r) { return (o << log_rows) + ((r ^ o) & row_mask); };
  unsigned xo[4];                                                // a lane's pieces of a step
#pragma unroll
  for (int c = 0; c < 4; ++c) xo[c] = (unsigned)place(SWAP ? c * 4 + quad : quad * 4 + c, l16) * 16u;

  // ---- where operands lie: a place that the wavefront shares, and 32 bits of the lane ----
  const int n1 = n0 < q.n ? n0 : q.n - 1, row = n0 + l16 < q.n ? l16 : q.n - 1 - n1;
  const size_t weight = (size_t)(there ? e : 0) * (p.gated ? 2 : 1) * q.n + (up ? q.n : 0) + n1;
  const char* const wt = (const char*)q.w + weight * pitch;
  const char* const st = (const char*)p.scale + weight * groups * S;
  const char* const bt = (const char*)p.bias + weight * groups * S;
  const unsigned wo = (unsigned)row * (unsigned)pitch + (unsigned)quad * 16u, go = (unsigned)row * (unsigned)groups * S;

  const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
  f32x4 acc = zero;
  typedef Groups<2 * kPer, S> Pair;                              // of two steps: quad i has steps 2 i and 2 i + 1 of a block
  u32x4 w[8];
  Pair scale, bias;
#pragma unroll
  for (int i = 0; i < Pair::kWords; ++i) bias.v[i] = 0u;
  const float shift = p.bias ? -16.0f : -24.0f;
  unsigned sixteen = F16 ? 0x4c004c00u : 0x41804180u;
  asm("" : "+v"(sixteen));
  const bf16x8 ones = __builtin_bit_cast(bf16x8, F16 ? u32x4{0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u} : u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});

  // A wavefront's steps of a pass: the first one's place in the row, how many there are from there on.
  auto share = [&](int base, int& from, int& left) {
    const int count = steps - base < per_pass ? steps - base : per_pass, s0 = (count * slice) >> p.log_split;
    from = base + s0;
    left = ((count * (slice + 1)) >> p.log_split) - s0;
  };
  auto load_w = [&](u32x4& to_w, int s) __attribute__((always_inline)) { __builtin_memcpy(&to_w, wt + (size_t)s * 64 + wo, 16); };
  // Groups of a block's steps.  The row's last step may be the first of a pair: then it is read as the second one of the pair before.
  auto load_groups = [&](int from, int here) __attribute__((always_inline)) {
    const int i = 2 * quad < here ? 2 * quad : here - 1;
    if (steps > 1) {
      const bool end = from + i + 1 == steps;
      const unsigned at = (unsigned)(from + i - (end ? 1 : 0)) * (kPer * S) + go;
      scale.load(st + at);
      if (p.bias) bias.load(bt + at);
      scale.drop_half(end);
      if (p.bias) bias.drop_half(end);
    } else {
      scale.load_part(st + go, kPer);
      if (p.bias) bias.load_part(bt + go, kPer);
    }
  };
  float sum[2 * kPer];                                           // of a block's groups of x, in the scales' order
  auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < 2 * kPer; ++g) sum[g] = 0.0f;
  };
  // step I of a block, x's pieces given by `piece`
  auto multiply = [&](auto step, auto piece) __attribute__((always_inline)) {
    constexpr int I = decltype(step)::value;
    if (SWAP) transpose4(w[I]);
    f32x4 t, one;
    each<4>([&](auto c_) __attribute__((always_inline)) {
      constexpr int c = decltype(c_)::value, g = (I & 1) * kPer + c / kIn;
      constexpr bool fresh = c % kIn == 0;
      const bf16x8 xv = piece(c);
      one = mm<F16>(ones, xv, fresh ? zero : one);
      t = mm<F16>(xv, widen<F16>(w[I][c], sixteen), fresh ? zero : t);
      if constexpr (c % kIn == kIn - 1) {
        sum[g] = quad == I >> 1 ? one[0] : sum[g];
        const float f = Pair::template value<F16>(of_quad<(I >> 1)>(scale.v[g * S / 4]), g);
#pragma unroll
        for (int v = 0; v < 4; ++v) acc[v] = fmaf(f, t[v], acc[v]);
      }
    });
  };
  // the part of a block that goes by the sums of x, as far as its steps go
  auto shifts = [&](int here) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < 2 * kPer; ++g) {
      const bool mine = 2 * quad + (g >= kPer ? 1 : 0) < here;
      const float off = mine ? fmaf(shift, Pair::template value<F16>(scale.v[g * S / 4], g), Pair::template value<F16>(bias.v[g * S / 4], g)) : 0.0f;
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(sum[g], off, acc, 0, 0, 0);
    }
  };

  // A thread brings up to eight pieces of a pass, of one row or (16 rows, eight wavefronts or fewer) of several; those past the end repeat the last one.
  const int beside = waves * 64 >> log_rows > 64 ? waves * 64 >> log_rows : 64, log_each = waves * 64 >> log_rows >= 64 ? 3 : 31 - __builtin_clz(waves * 512 >> (log_rows + 6));
  const int row0 = wave & row_mask, piece0 = (wave >> log_rows) * 64 + lane;
  int from = 0, left = 0;
  for (int base = 0; base < steps; base += per_pass) {
    const int count = steps - base < per_pass ? steps - base : per_pass, last = count * 16 - 1;
    if (base > 0) __syncthreads();
    u32x4 v[4];
    int o[4], r[4];
    auto fetch = [&](int h) __attribute__((always_inline)) {      // four pieces
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int at = piece0 + ((4 * h + u) & ((1 << log_each) - 1)) * beside, x_row = row0 + ((4 * h + u) >> log_each) * waves;
        o[u] = at < last ? at : last;
        r[u] = x_row < rows ? x_row : rows - 1;
        __builtin_memcpy(&v[u], xb + ((size_t)r[u] * q.x_pitch + (size_t)base * 128) * 2 + (unsigned)o[u] * 16u, 16);
      }
    };
    auto put = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < 4; ++u) smem[place(o[u], r[u])] = __builtin_bit_cast(u32x4, reorder(v[u]));
    };
    fetch(0);
    if (log_each < 3 || last >= 4 * beside) {
      put();
      fetch(1);
    }
    if (base == 0) {                                             // (x is asked for before the first weights: it is needed first)
      share(0, from, left);
      if (left > 0) {
        const int here = left < 8 ? left : 8;
        load_groups(from, here);
#pragma unroll
        for (int i = 0; i < 8; ++i) load_w(w[i], from + (i < here ? i : here - 1));
      }
    }
    put();
    __syncthreads();
    // ---- this wavefront's blocks of it ----
    while (left > 0) {
      const int here = left < 8 ? left : 8;
      int next = from + here, next_left = left - here;
      if (next_left == 0 && base + per_pass < steps) share(base + per_pass, next, next_left);
      const bool more = next_left > 0;
      if (!more) next = from;                                    // (what is requested then is not used)
      const int next_here = !more ? here : next_left < 8 ? next_left : 8;
      const char* const at = (const char*)smem + ((unsigned)(from - base) << (log_rows + 8));
      clear();
      each<8>([&](auto i_) __attribute__((always_inline)) {
        constexpr int i = decltype(i_)::value;
        if (i < here) {
          const char* const to_x = at + ((unsigned)i << (log_rows + 8));
          multiply(i_, [&](int c) __attribute__((always_inline)) { return *reinterpret_cast<const bf16x8*>(to_x + xo[c]); });
        }
        load_w(w[i], next + (i < next_here ? i : next_here - 1));
        __builtin_amdgcn_sched_barrier(0);
      });
      shifts(here);
      load_groups(next, next_here);
      left -= here;
      from = next;
      if (left == 0) {                                           // (the next pass's, if there is one)
        left = next_left;
        break;
      }
    }
  }
  // channels behind the last whole step: the last slice's; zeros for those that are not there
  const int rest = q.k & 127;
  if (rest && there && slice == split - 1) {
    const char* const at = xb + (size_t)(l16 < rows ? l16 : rows - 1) * q.x_pitch * 2 + (size_t)steps * 256 + quad * 16;
    const unsigned group = (unsigned)steps * (kPer * S) + go;
    scale.load_part(st + group, groups - steps * kPer);
    if (p.bias) bias.load_part(bt + group, groups - steps * kPer);
    w[0] = u32x4{0u, 0u, 0u, 0u};
    if (quad * 32 < rest) load_w(w[0], steps);
    clear();
    multiply(Count<0>(), [&](int c) __attribute__((always_inline)) {
      u32x4 v = {0u, 0u, 0u, 0u};
      if (c * 32 < rest) __builtin_memcpy(&v, at + c * 64, 16);
      return reorder(v);
    });
    shifts(1);
  }

  // ---- the slices' sums, in order; lane: weight row l % 16, rows 4 (l / 16) + 0..3 ----
  f32x4* const sums = reinterpret_cast<f32x4*>(smem);            // [tiles][slices][64]
  if (split > 1 || p.gated) {
    __syncthreads();
    sums[wave * 64 + lane] = acc;
    __syncthreads();
  }
  if (slice != 0 || up) return;
  auto sum_of = [&](int t) {
    f32x4 v = sums[(t << p.log_split) * 64 + lane];
    for (int k = 1; k < split; ++k) v += sums[((t << p.log_split) + k) * 64 + lane];
    return v;
  };
  f32x4 v = split > 1 || p.gated ? sum_of(tile) : acc;
  if (p.gated) {
    const f32x4 u = sum_of(to + tile);
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = gated(v[c], u[c], q.activation);
  }
  const int n = n0 + l16;
  if (n >= q.n) return;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (quad * 4 + c < rows) store_as(q.y, (size_t)(first + quad * 4 + c) * q.y_pitch + n, q.y_dtype, v[c]);
}

template <int G, bool F16, int S>
int launch(W4Params p, hipStream_t stream) {
  const GroupedParams& q = p.g;
  const long long tails = q.experts + 1 < q.rows ? q.experts + 1 : q.rows;        // tiles of rows that are not full, at most
  const long long tiles_m = !q.offsets ? (q.rows + 15) / 16 : q.rows / 16 + tails < q.rows ? q.rows / 16 + tails : q.rows;
  const long long work = tiles_m * ((q.n + 15) / 16) * (p.gated ? 2 : 1);         // tiles of rows of x and of the weight
  const int steps = q.k / 128;
  // Tiles of a workgroup share x's way through LDS: as few as leave a workgroup to a CU (with up to four rows of x, two).  Four wavefronts where
  // there is plenty of work or little to divide.  Measured, us 1 / 2 / 4 tiles with 4 wavefronts, then with 8, rows x n x k: 1 x 2048 x
  // 7168 10 / 15 / 25, 9.6 / 12 / 19; 4 x 16384 x 7168 26 / 24 / 30, 30 / 23 / 23; 48 x 2048 x 7168 27 / 26 / 32, 30 / 21 / 24; 48 x 4096 x 4096 26 /
  // 20 / 20, 30 / 21 / 15; 8 x 2048 x 2048 7.8 / 8.5 / 11, 9.2 / 9.3 / 9.9; 16 x 8192 x 2048 13 / 11 / 12, 14 / 10 / 11; 16 x 16384 x 7168 50 / 35 /
  // 37, 60 / 33 / 28; 64 x 8192 x 8192 105 / 58 / 46, 117 / 64 / 39; 1024 x 1024 x 512 41 / 23 / 14, 61 / 44 / 24; 256 x 61 experts gated, 2 and 4
  // tiles: 269 / 243, 306 / 263.
  const bool thin = q.rows <= 4 && q.experts == 1;
  const int tiles = work > 512 && !thin ? 4 : work > 256 || p.gated ? 2 : 1;
  const int waves = work >= 4096 || steps * tiles < 32 ? 4 : 8;
  p.log_split = __builtin_ctz(waves / tiles);
  const int out = 16 * (p.gated ? tiles / 2 : tiles), parts = (q.n + out - 1) / out;
  if (int rc = check_tiles("w4_gemm", parts, 64 * waves)) return rc;
  constexpr long long kMostY = 65535;                            // (of a grid)
  for (long long t = 0; t < tiles_m; t += kMostY) {
    p.tile0 = (int)t;
    const dim3 grid((unsigned)parts, (unsigned)(tiles_m - t < kMostY ? tiles_m - t : kMostY));
    hipLaunchKernelGGL((w4_kernel<G, F16, S>), grid, dim3(64 * waves), (size_t)waves * kRoom, stream, p);
  }
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
  if (a.n > (is_gated ? CPPMEGA_MI355_GATED_MAX_OUTPUTS : CPPMEGA_MI355_GROUPED_MAX_SIZE))
    return fail(CPPMEGA_MI355_ERR_SHAPE, "w4_gemm: n=%d, at most 2^30 weight rows are served", a.n);
  // (a lane's place in a tile's rows is kept in 32 bits)
  if (a.k > CPPMEGA_MI355_W4_MAX_CHANNELS || a.x_pitch < 0 || a.x_pitch > CPPMEGA_MI355_W4_MAX_CHANNELS)
    return fail(CPPMEGA_MI355_ERR_SHAPE, "w4_gemm: k=%d and rows of x %lld apart, at most 2^24 are served", a.k, (long long)a.x_pitch);
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
  // Weights widened once for 64 rows, or once for 16 with eight times the wavefronts: the former from 32 rows to an expert on, where there is as much
  // work as makes up for its start, in tiles of 16 x 16 results.  Measured, us 64 / 16 rows, rows x n x k: 64 x 8192 x 8192 54 / 39, 64 x 16384 x
  // 4096 31 / 40, 64 x 4096 x 4096 27 / 16, 128 x 4096 x 4096 28 / 23, 256 x 4096 x 4096 29 / 36, 32 x 32768 x 2048 25 / 24, 512 x 8192 x 8192 135 / 229, 4096 x
  // 4096 x 4096 303 / 457; gated 512 x 16 experts x 1024 x 2048 25 / 32, 256 x 16 experts x 1024 x 7168 61 / 53.  Where the rule takes the slower one: 1024 x 1024
  // x 512 11 / 14.
  const double tiles = ((a.rows + 15) / 16 + (a.experts > 1 ? a.experts / 2 : 0)) * (((double)a.n * (is_gated ? 2 : 1) + 15) / 16);
  if (a.rows >= 32ll * a.experts && a.k >= 1024 && tiles >= 2560.0) return w4_tile_launch(p, a.group, f16, wide, stream);
  return a.group == 32 ? launch_group<32>(p, f16, wide, stream) : a.group == 64 ? launch_group<64>(p, f16, wide, stream) : launch_group<128>(p, f16, wide, stream);
}

}  // namespace cm

// Products grouped by expert for many rows (gfx950): 256 x 256 and 128 x 128 tiles, operands by the load unit into LDS.
//
// Needs rows that begin on 16 bytes and a contraction (and, where it is the slow axis, columns) in whole 16-byte pieces.
//
// LDS holds rings of stages of both operands, 128 or 64 bytes of contraction each, filled by global_load_lds as far ahead as there is room;
// two wavefronts on a SIMD, one barrier a stage, behind which the next stage's first operands are read under this one's last products.
// Rows that are not there repeat the last one and are not stored; contraction that is not there comes from a piece of zeros, for both
// operands (what lies behind a row may be NaN).  Each wavefront has
// every other 32 rows of the tile and multiplies as many of them as there are; one without rows only loads.  16-bit products by 32 x 32 x 16
// instructions; e4m3 by 16 x 16 x 128, a scale block each, whose sums are scaled and added while the matrix unit is at the next ones.
// That instruction aligns eight products to the largest of them and drops what lies below 2^-13 of it, whatever is left of the largest in the
// end: with two of 448^2 that cancel, six of 14 are lost.  Only bfloat16 results take it, whose rounding is a hundred times what it costs
// normally distributed codes (measured, K 128 to 7168: 1.5e-5 of the results' root mean square, beside 1.65e-3; the exact products of the
// register kernel take four times as long); results of more bits are not made here.
// Pieces are 16 bytes; in LDS
//   contraction contiguous: [row][pieces], piece c of row r in place c ^ fold(r);
//   contraction slow: [step][pieces of 8 channels], piece c of step s in place c ^ 4 (s % 4), read by the transposing load.
// (No bank conflicts in either: counted.)
//
// Measured, us (TFLOP/s): 16384 rows of 32 experts, 4096 x 2048 bf16 308 (890); of one expert 248 (1110), and 4096 x 8192 833 (1320), where a library's
// product of that size reaches 1390: at 1.3 PFLOP/s the clock is down at 1.7 GHz, power is the bound, and neither deeper rings nor other orders
// of loads change it.  What short contractions lose: 10 to 12 us a tile for its first loads and for stores that all CUs send at once; persistent
// workgroups with the next tile's first stages under the stores were not faster, and tiles of few rows after all others 5 % slower (the weights are
// read twice).  Both gradients, 8192 rows of 16 experts, 4096 x 2048 bf16, in one launch 329 (835); one after the other 375: the
// rows' 320 tiles leave 192 of 512 places empty, and a gradient's contraction is 512 rows.
// e4m3, 4096 x 7168 of 32 experts 600 (1600), 4096 x 8192 of one 510 (2150): of a SIMD's cycles the products take 0.41 and the scaling's multiply-adds
// (one per result and block: none to spare) 0.30, at 1.9 GHz; its two wavefronts could be at the one and the other at once, but pass the same barriers and
// do the same at the same time (a wavefront waits 0.28 of its own cycles).  The multiply-adds spread between single products changed nothing.

#include <type_traits>

#include "grouped_gemm.h"

namespace cm {
namespace {

__device__ __align__(64) const unsigned char zeros[64] = {};

// HIGH: 256 x 256 tiles, eight wavefronts of 128 x 64, one workgroup to a CU.  Otherwise 128 x 128, four of 64 x 64, two to a CU.
template <int OP, int DT, bool HIGH>
struct Shape {
  static constexpr bool FP8 = DT == CPPMEGA_MI355_E4M3, F16 = DT == CPPMEGA_MI355_F16;
  static constexpr bool TR = OP == kWeightsGrad, TQ = OP != kRows;      // the contraction is the operand's slow axis
  static constexpr int BM = HIGH ? 256 : 128, BN = BM, WN = HIGH ? 4 : 2, kWaves = 2 * WN;
  static constexpr int kHeight = BM / 2, kWidth = BN / WN;              // of a wavefront
  // Bytes of contraction in a stage, and how many stages of each operand LDS holds.  Pieces of 64 bytes of a row arrive at half the
  // rate of whole lines (5 % of a large product); of the slow axis a stage has whole rows of the tile either way, and more of them on
  // their way are worth 7 %.
  static constexpr int KB = FP8 || !TQ ? 128 : 64;
  static constexpr int RS = KB == 64 ? (HIGH ? 5 : 4) : FP8 || !HIGH ? 2 : 3, QS = KB == 64 ? RS : 2;
  static constexpr int BYTES = FP8 ? 1 : 2, STEP = KB / BYTES;
  static constexpr int RL = BM * KB / 1024 / kWaves, QL = BN * KB / 1024 / kWaves, L = RL + QL + (FP8 ? 1 : 0);   // load instructions per wavefront and stage
  static constexpr int kR = BM * KB, kQ = BN * KB, kS = FP8 ? kWaves * 256 : 0;
  static constexpr int kQat = RS * kR, kSat = kQat + QS * kQ, kLds = kSat + QS * kS;            // where columns and scales begin
  // the place of piece c of a row among its row's pieces is c ^ fold(row): sixteen rows with one piece lie in different banks
  static __device__ __forceinline__ int fold(int row) { return KB == 128 ? (row >> 1) & 7 : (row >> 2) & 3; }
};

template <int N>
using Count = std::integral_constant<int, N>;

// Tile `block` of a product (of the launch's order, or none: every XCD's blocks are counted up to the same number), in S::kLds bytes of LDS.
// `cut`: the last round's tiles in parts.
template <int OP, int DT, bool HIGH>
__device__ __forceinline__ void tile_of(const GroupedParams& p, const int block, u32x4* const smem, const bool cut) {
  typedef Shape<OP, DT, HIGH> S;                                 // (inlined throughout: a call would put the sums into memory)
  constexpr bool FP8 = S::FP8, F16 = S::F16, TR = S::TR, TQ = S::TQ;
  constexpr int BYTES = S::BYTES, STEP = S::STEP, BM = S::BM, BN = S::BN, RS = S::RS, QS = S::QS, RL = S::RL, QL = S::QL, L = S::L, KB = S::KB;
  static_assert(S::kLds >= (kMaxExperts + 2) * (int)sizeof(int), "the tiles' table lies where the stages are later");
  int* const starts = reinterpret_cast<int*>(smem);
  char* const lds = reinterpret_cast<char*>(smem);
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = (wave % S::WN) * S::kWidth, upper = wave / S::WN;   // a wavefront's columns; every other 32 rows are its rows

  // ---- which tile: every XCD takes one run of the order, which goes through the experts; of each, up to four row tiles share the
  // columns that pass, so that an expert's weight leaves memory once (groups of four rows of tiles whatever their experts: 5 % slower) ----
  const int cols_c = OP == kRows ? p.n : p.k;
  const int tiles_n = (cols_c + BN - 1) / BN;
  const int per_expert = OP == kWeightsGrad ? (p.n + BM - 1) / BM : 0;
  int e, m0, n0, part_rows = BM;
  {
    const int xcd = block & 7, at = block >> 3;
    int local, high, part = 0;                                   // tile of the expert, its rows of tiles
    if (OP == kWeightsGrad) {
      // (experts differ in length here, not in tiles: every XCD takes an eighth of each expert; whole experts to an XCD left CUs idle
      // for a third of the time)
      const int share = (per_expert * tiles_n + 7) / 8;
      e = at / share;
      local = xcd * share + at - e * share;
      if (local >= per_expert * tiles_n) return;
      high = per_expert;
    } else {
      const int total = fill_tiles<BM>(p, starts) * tiles_n, q = total >> 3, r = total & 7;
      // A last round that leaves half of the XCD's CUs idle or more is made of halves or quarters of its tiles (128 or 64 rows: 0.67 and
      // 0.5 of a tile's time).
      constexpr int kSlots = HIGH ? 32 : 64, kParts = BM / 64;
      const int mine = q + (xcd < r ? 1 : 0), last = mine % kSlots, from = mine - last;
      const int parts = !cut ? 1 : last * 4 <= kSlots && kParts >= 4 ? 4 : last * 2 <= kSlots ? 2 : 1;
      if (at >= from + last * parts) return;
      const int tile = at < from ? at : from + (at - from) / parts;
      if (at >= from) {
        part = (at - from) % parts;
        part_rows = BM / parts;
      }
      const int id = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + tile;
      e = expert_of_tile(p, starts, id / tiles_n);
      local = id - starts[e] * tiles_n;
      high = starts[e + 1] - starts[e];
    }
    const int groups = (high + 3) / 4, step = (high + groups - 1) / groups;       // rows of tiles in a group
    const int group = local / (step * tiles_n), in = local - group * step * tiles_n;
    const int height = high - group * step < step ? high - group * step : step;
    const int nt = in / height;
    n0 = nt * BN;
    m0 = (group * step + in - nt * height) * BM + part * part_rows;
  }
  const int lo = __builtin_amdgcn_readfirstlane((int)offset_of(p, e));
  const int hi = __builtin_amdgcn_readfirstlane(e < p.experts ? (int)offset_of(p, e + 1) : (int)p.rows);
  const int tokens = hi > lo ? hi - lo : 0;
  m0 = __builtin_amdgcn_readfirstlane(m0);
  n0 = __builtin_amdgcn_readfirstlane(n0);
  const int contraction = OP == kWeightsGrad ? tokens : (e == p.experts ? 0 : (OP == kRows ? p.k : p.n));
  const int rows_left = (OP == kWeightsGrad ? p.n : tokens) - m0, rows_here = rows_left < part_rows ? rows_left : part_rows, cols_here = cols_c - n0;
  if (rows_here <= 0) return;                                   // (a part behind the expert's last row)
  const int stages = (contraction + STEP - 1) / STEP, whole = contraction / STEP;
  const long long w_pitch = OP == kWeightsGrad ? p.w_pitch : p.k;

  // ---- loads ----
  const char* xb = (const char*)p.x + ((size_t)lo * p.x_pitch + (TR ? (size_t)m0 : (size_t)m0 * p.x_pitch)) * BYTES;
  const char* wb = (const char*)p.w + ((OP == kWeightsGrad ? (size_t)lo * p.w_pitch : (size_t)(e < p.experts ? e : 0) * p.n * p.k) + (TQ ? (size_t)n0 : (size_t)n0 * p.k)) * BYTES;
  const long long x_step = TR ? p.x_pitch * STEP * BYTES : KB, w_step = TQ ? w_pitch * STEP * BYTES : KB;
  unsigned xoff[RL], woff[QL], soff = 0;
  // where a lane's piece of load instruction u of an operand lies, and how far along the contraction that is
  constexpr int PIECES = KB / 16;                                // of a row in a stage
  auto piece_of = [&](bool transposed, int u, int limit, long long pitch) -> unsigned {
    if (!transposed) {
      const int row = u * (64 / PIECES) + lane / PIECES, c = (lane % PIECES) ^ S::fold(row);
      return (unsigned)((row < limit ? row : limit - 1) * pitch * BYTES) + (unsigned)c * 16u;
    }
    const int step = u * (512 / BM) + lane / (BM / 8), c = (lane % (BM / 8)) ^ ((step & 3) << 2);
    return (unsigned)(step * pitch * BYTES) + (unsigned)(c * 8 < limit ? c : (limit - 1) >> 3) * 16u;
  };
  auto along = [&](bool transposed, int u) {
    return transposed ? u * (512 / BM) + lane / (BM / 8) : ((lane % PIECES) ^ S::fold(u * (64 / PIECES) + lane / PIECES)) * (16 / BYTES);
  };
#pragma unroll
  for (int i = 0; i < RL; ++i) xoff[i] = piece_of(TR, wave * RL + i, rows_here, p.x_pitch);
#pragma unroll
  for (int i = 0; i < QL; ++i) woff[i] = piece_of(TQ, wave * QL + i, cols_here, w_pitch);
  const char* sb = nullptr;
  unsigned s_step = 0;
  if constexpr (FP8) {
    // half of the wavefronts bring the scales of 64 rows each, the others those of the columns' blocks
    const int blocks_k = (p.k + 127) / 128, blocks_n = (p.n + 127) / 128;
    if (wave < BM / 64) {
      const int row = wave * 64 + lane;
      sb = (const char*)(p.x_scale + (size_t)(lo + m0) * (p.x_scale_block ? blocks_k : 1));
      soff = (unsigned)(row < rows_here ? row : rows_here - 1) * (p.x_scale_block ? (unsigned)blocks_k * 4u : 4u);
      s_step = p.x_scale_block ? 4u : 0u;
    } else {
      const int b = n0 / 128 + (BN > 128 ? lane & 1 : 0);
      sb = (const char*)(p.w_scale + (size_t)(e < p.experts ? e : 0) * blocks_n * blocks_k);
      soff = (unsigned)(b < blocks_n ? b : blocks_n - 1) * (unsigned)blocks_k * 4u;
      s_step = 4u;
    }
  }
  const unsigned lds_base = (unsigned)(size_t)(lds_void*)smem;
  auto load16 = [&](const char* base, unsigned off, unsigned to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(off), "s"(base) : "memory", "m0");
  };
  auto load16_at = [&](const char* at, unsigned to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(at) : "memory", "m0");
  };
  auto load4 = [&](const char* base, unsigned off, unsigned to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(to), "v"(off), "s"(base) : "memory", "m0");
  };
  int next_r = 0, next_q = 0;                                   // stages of rows and of columns to be requested next
  unsigned r_slot = lds_base, q_slot = lds_base + S::kQat, s_slot = lds_base + S::kSat;
  // Requests instruction i of a stage: the columns' (and scales') first, then the rows', which may be a stage further on.  MORE:
  // whole stages.  Otherwise the last one, of which a part may not be there, or one behind it: pieces of zeros (no branch here or in the
  // loops below: the compiler moves products across branches, away from the reads that they cover).
  auto issue = [&](auto more, int from, int to) __attribute__((always_inline)) {
    constexpr bool MORE = decltype(more)::value;
#pragma unroll
    for (int i = 0; i < L; ++i) {
      if (i < from || i >= to) continue;
      if (i < L - RL) {
        if (i < QL) {
          const int u = wave * QL + i;
          unsigned off = woff[i < QL ? i : 0];
          if (MORE) {
            load16(wb, off, q_slot + (unsigned)(u * 1024));
          } else {
            asm("" : "+v"(off));                                // (the address is made here, not kept in registers throughout)
            load16_at(next_q * STEP + along(TQ, u) < contraction ? wb + off : (const char*)zeros, q_slot + (unsigned)(u * 1024));
          }
        } else {
          const bool there = MORE || next_q < stages;
          load4(there ? sb : (const char*)zeros, there ? soff : 0u, s_slot + (unsigned)(wave * 256));
        }
        if (i == L - RL - 1) {
          wb += w_step;
          sb += s_step;
          ++next_q;
          q_slot = q_slot + S::kQ == lds_base + S::kSat ? lds_base + S::kQat : q_slot + S::kQ;
          if (FP8) s_slot = s_slot + S::kS == lds_base + S::kLds ? lds_base + S::kSat : s_slot + S::kS;
        }
      } else {
        const int u = wave * RL + i - (L - RL);
        unsigned off = xoff[i < L - RL ? 0 : i - (L - RL)];
        if (MORE) {
          load16(xb, off, r_slot + (unsigned)(u * 1024));
        } else {
          asm("" : "+v"(off));
          load16_at(next_r * STEP + along(TR, u) < contraction ? xb + off : (const char*)zeros, r_slot + (unsigned)(u * 1024));
        }
        if (i == L - 1) {
          xb += x_step;
          ++next_r;
          r_slot = r_slot + S::kR == lds_base + S::kQat ? lds_base : r_slot + S::kR;
        }
      }
    }
  };
  typedef std::integral_constant<bool, true> Whole;
  typedef std::integral_constant<bool, false> Part;
  if (OP != kWeightsGrad) __syncthreads();                       // (the tiles' table has been read)
  if (stages > 0) {
#pragma unroll
    for (int s = 0; s < RS; ++s) {
      if (s < RS - QS) issue(Part(), L - RL, L);
      else if (s < whole) issue(Whole(), 0, L);
      else issue(Part(), 0, L);
    }
    // rows 0 .. RS - QS, columns 0 have arrived
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((QS - 1) * L) : "memory");
  }
  const int steady = whole - RS;                                 // stages while whose products whole ones are requested
  // between a stage's last operand reads and its last products: the next stage has arrived, and everybody has read this one
  constexpr int kYounger = (QS - 2) * L + (RS > QS ? RL : 0);    // instructions behind those of the next stage
  auto turn = [&] { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kYounger) : "memory"); };
  const int runs = rows_here - upper * 32 > 0 ? (rows_here - upper * 32 + 63) / 64 : 0;   // of 32 rows that a wavefront has, the last one in part
  auto follow = [&]() __attribute__((always_inline)) {            // a wavefront without rows: its loads only
    for (int s = 0; s + 1 < stages; ++s) {
      turn();
      if (s < steady) issue(Whole(), 0, L);
      else issue(Part(), 0, L);
    }
  };
  int r_at = 0, q_at = S::kQat, s_at = S::kSat;                  // where the stage that is multiplied lies
  auto r_after = [&] { return r_at + S::kR == S::kQat ? 0 : r_at + S::kR; };
  auto q_after = [&] { return q_at + S::kQ == S::kSat ? S::kQat : q_at + S::kQ; };
  auto s_after = [&] { return s_at + S::kS == S::kLds ? S::kSat : s_at + S::kS; };
  const size_t row0 = OP == kWeightsGrad ? (size_t)e * p.n + m0 : (size_t)lo + m0;
  const long long y_pitch = OP == kWeightsGrad ? p.k : p.y_pitch;
  // 8 (16-bit) or 4 (float32) values of a row, as far as the columns go
  auto store = [&](int row, int col, const float* v, int count) __attribute__((always_inline)) {
    if (row >= rows_here || col >= cols_here) return;
    const size_t at = (row0 + row) * y_pitch + n0 + col;
    if (col + count <= cols_here) {
      if (p.y_dtype == CPPMEGA_MI355_F32) {
        __builtin_memcpy((float*)p.y + at, v, 4 * count);
      } else {
        unsigned r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (2 * i < count) r[i] = p.y_dtype == CPPMEGA_MI355_F16 ? pack_f16(v[2 * i], v[2 * i + 1]) : pack_bf16(v[2 * i], v[2 * i + 1]);
        __builtin_memcpy((unsigned short*)p.y + at, r, 2 * count);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < count && col + i < cols_here) store_as(p.y, at + i, p.y_dtype, v[i]);
    }
  };

  if constexpr (!FP8) {
    constexpr int TI = S::kHeight / 32, TJ = S::kWidth / 32;        // 32 x 32 tiles of the wavefront
    const int l32 = lane & 31, half = lane >> 5, l16 = lane & 15;
    constexpr int KS = KB / 32;                                 // 16 steps of contraction at a time
    int rat[TR ? TI : KS], qat[TQ ? TJ : KS];                     // where a lane reads: per tile (transposing), or per 16 steps
    if (TR) {
#pragma unroll
      for (int i = 0; i < TI; ++i) {
        const int col = i * 64 + upper * 32 + (lane & 16) + (l16 & 3) * 4;
        rat[i] = (half * 8 + (l16 >> 2)) * (BM * 2) + ((col >> 3) ^ ((l16 >> 2) << 2)) * 16 + (col & 4) * 2;
      }
    } else {
#pragma unroll
      for (int k = 0; k < KS; ++k) rat[k] = (upper * 32 + l32) * KB + ((2 * k + half) ^ S::fold(l32)) * 16;
    }
    if (TQ) {
#pragma unroll
      for (int j = 0; j < TJ; ++j) {
        const int col = wn + j * 32 + (lane & 16) + (l16 & 3) * 4;
        qat[j] = (half * 8 + (l16 >> 2)) * (BN * 2) + ((col >> 3) ^ ((l16 >> 2) << 2)) * 16 + (col & 4) * 2;
      }
    } else {
#pragma unroll
      for (int k = 0; k < KS; ++k) qat[k] = (wn + l32) * KB + ((2 * k + half) ^ S::fold(l32)) * 16;
    }
    auto transposed = [&](int at, int pitch4) -> bf16x8 {       // eight steps of a lane's channel
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds + at)));
      const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds + at + pitch4)));
      return __builtin_bit_cast(bf16x8, u32x4{a[0], a[1], b[0], b[1]});
    };
    bf16x8 r[2][TI], q[2][TJ];
    auto read_ahead = [&](auto n, int rows, int cols, int ks) __attribute__((always_inline)) {
      const int to = ks & 1;
#pragma unroll
      for (int j = 0; j < TJ; ++j) q[to][j] = TQ ? transposed(cols + qat[j] + ks * 16 * BN * 2, 4 * BN * 2) : *reinterpret_cast<const bf16x8*>(lds + cols + qat[TQ ? 0 : ks] + j * 32 * KB);
#pragma unroll
      for (int i = 0; i < decltype(n)::value; ++i) r[to][i] = TR ? transposed(rows + rat[i] + ks * 16 * BM * 2, 4 * BM * 2) : *reinterpret_cast<const bf16x8*>(lds + rows + rat[TR ? 0 : ks] + i * 64 * KB);
      __builtin_amdgcn_sched_barrier(0);
    };
    f32x16 acc[TI][TJ];
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
      for (int j = 0; j < TJ; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.0f;
    // products of one 16 steps of the first n of the rows' tiles; between them load instructions from .. (all at once, the wavefronts
    // stood still until the load unit's queue had room)
    auto multiply = [&](auto n, int b, auto more, int from) __attribute__((always_inline)) {
      constexpr int N = decltype(n)::value;
#pragma unroll
      for (int i = 0; i < N; ++i) {
#pragma unroll
        for (int j = 0; j < TJ; ++j) {
          if constexpr (F16) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, q[b][j]), __builtin_bit_cast(f16x8, r[b][i]), acc[i][j], 0, 0, 0);
          else acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(q[b][j], r[b][i], acc[i][j], 0, 0, 0);
        }
        if (from >= 0) {
          __builtin_amdgcn_sched_barrier(0);
          issue(more, L * i / N, L * (i + 1) / N);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    auto stage = [&](auto n, auto more) __attribute__((always_inline)) {
      const int rows = r_after(), cols = q_after();
#pragma unroll
      for (int ks = 0; ks + 1 < KS; ++ks) {
        read_ahead(n, r_at, q_at, ks + 1);
        multiply(n, ks & 1, more, -1);
      }
      turn();
      read_ahead(n, rows, cols, 0);
      multiply(n, (KS - 1) & 1, more, 0);
      r_at = rows;
      q_at = cols;
    };
    auto all = [&](auto n) __attribute__((always_inline)) {
      read_ahead(n, r_at, q_at, 0);
      int s = 0;
      for (; s < steady; ++s) stage(n, Whole());
      for (; s + 1 < stages; ++s) stage(n, Part());
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if (ks + 1 < KS) read_ahead(n, r_at, q_at, ks + 1);
        multiply(n, ks & 1, Part(), -1);
      }
    };
    if (stages > 0) {
      if (runs == 0) follow();
      else if (runs >= TI || OP == kWeightsGrad) all(Count<TI>());
      else if (runs == 1) all(Count<1>());
      else if (runs == 2) all(Count<(TI > 2 ? 2 : 1)>());
      else all(Count<(TI > 3 ? 3 : 1)>());
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");            // (what was requested behind the end still writes to LDS)
    // lane: row l % 32, columns 8 q + 4 (l / 32) + 0..3; the halves change places so that a lane has 8 columns in a run
    if (runs > 0) {
#pragma unroll
      for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float v[8];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const u32x2 x = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[i][j][h * 8 + c]), __float_as_uint(acc[i][j][h * 8 + 4 + c]), false, false);
              v[c] = __uint_as_float(x[0]);
              v[4 + c] = __uint_as_float(x[1]);
            }
            store(i * 64 + upper * 32 + l32, wn + j * 32 + h * 16 + half * 8, v, 8);
          }
    }
  } else {
    constexpr int TI = S::kHeight / 16, TJ = S::kWidth / 16;        // 16 x 16 tiles of the wavefront, a whole 128-channel block an instruction
    const int l16 = lane & 15, quad = lane >> 4, f = (l16 >> 1) & 7;
    const int rat[2] = {(upper * 32 + l16) * 128 + (quad ^ f) * 16, (upper * 32 + l16) * 128 + ((quad + 4) ^ f) * 16};
    const int qat[2] = {(wn + l16) * 128 + (quad ^ f) * 16, (wn + l16) * 128 + ((quad + 4) ^ f) * 16};
    const int xsat = (upper * 32 + l16) * 4, wsat = BM / 64 * 256 + (wn >> 7) * 4;
    auto operand = [&](int a, int b) -> i32x8 {
      const u32x4 x = *reinterpret_cast<const u32x4*>(lds + a), y = *reinterpret_cast<const u32x4*>(lds + b);
      i32x8 o;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o[i] = (int)x[i];
        o[4 + i] = (int)y[i];
      }
      return o;
    };
    f32x4 acc[TI][TJ];
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
      for (int j = 0; j < TJ; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    i32x8 q[TJ], r[2];
    float sx[TI], sw;
    auto read_q = [&](int from, int j) { q[j] = operand(from + qat[0] + j * 2048, from + qat[1] + j * 2048); };
    auto row_of = [](int i) { return (i >> 1) * 64 + (i & 1) * 16; };   // where the rows' tile i begins
    auto read_r = [&](int from, int i) { r[i & 1] = operand(from + rat[0] + row_of(i) * 128, from + rat[1] + row_of(i) * 128); };
    auto read_scales = [&](auto n, int from) {
#pragma unroll
      for (int i = 0; i < decltype(n)::value; ++i) sx[i] = *reinterpret_cast<const float*>(lds + from + xsat + row_of(i) * 4);
      sw = *reinterpret_cast<const float*>(lds + from + wsat);
    };
    // a block's products are scaled and added while the matrix unit is at the next ones
    f32x4 t[2][TJ];
    auto product = [&](int i, int j) {
      const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
      t[i & 1][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(q[j], r[i & 1], zero, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
    };
    auto add = [&](int i) {
      const float s = sx[i] * sw;
#pragma unroll
      for (int j = 0; j < TJ; ++j)
#pragma unroll
        for (int v = 0; v < 4; ++v) acc[i][j][v] = fmaf(s, t[i & 1][j][v], acc[i][j][v]);
    };
    // the first n of the rows' tiles (an even number) but the last; load instructions from .. between them, a share to a group of products
    auto products = [&](auto n, auto more, int from) __attribute__((always_inline)) {
      constexpr int N = decltype(n)::value, PER = (L + N - 1) / N;
#pragma unroll
      for (int i = 0; i < N - 1; ++i) {
        read_r(r_at, i + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < TJ; ++j) product(i, j);
        __builtin_amdgcn_sched_barrier(0);
        if (from >= 0 && from + PER * i < L) issue(more, from + PER * i, from + PER * i + PER < L ? from + PER * i + PER : L);
        if (i > 0) add(i - 1);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    // between a stage and the next: the last rows' products, and the next operands as soon as their registers are free
    auto pass = [&](auto n, auto more) __attribute__((always_inline)) {
      constexpr int N = decltype(n)::value, PER = (L + N - 1) / N;
      const int rows = r_after(), cols = q_after();
      turn();
      read_r(rows, 0);
#pragma unroll
      for (int j = 0; j < TJ; ++j) {
        product(N - 1, j);
        __builtin_amdgcn_sched_barrier(0);
        read_q(cols, j);
        __builtin_amdgcn_sched_barrier(0);
      }
      issue(more, 0, PER);
      add(N - 2);
      add(N - 1);
      s_at = s_after();
      read_scales(n, s_at);
      __builtin_amdgcn_sched_barrier(0);
      r_at = rows;
      q_at = cols;
    };
    auto all = [&](auto n) __attribute__((always_inline)) {
      constexpr int N = decltype(n)::value, PER = (L + N - 1) / N;
#pragma unroll
      for (int j = 0; j < TJ; ++j) read_q(q_at, j);
      read_r(r_at, 0);
      read_scales(n, s_at);
      products(n, Part(), -1);
      int s = 0;
      for (; s < steady; ++s) {
        pass(n, Whole());
        products(n, Whole(), PER);
      }
      for (; s + 1 < stages; ++s) {
        pass(n, Part());
        products(n, Part(), PER);
      }
#pragma unroll
      for (int j = 0; j < TJ; ++j) product(N - 1, j);
      add(N - 2);
      add(N - 1);
    };
    if (stages > 0) {
      if (runs == 0) follow();
      else if (runs >= TI / 2) all(Count<TI>());
      else if (runs == 1) all(Count<2>());
      else if (runs == 2) all(Count<(TI > 4 ? 4 : 2)>());
      else all(Count<(TI > 6 ? 6 : 2)>());
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    // lane: row l % 16, columns 4 (l / 16) + 0..3; two tiles' quarters change places so that a lane has 8 columns in a run
    if (runs > 0) {
#pragma unroll
      for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; j += 2) {
          float v[8];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const u32x2 x = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[i][j][c]), __float_as_uint(acc[i][j + 1][c]), false, false);
            v[c] = __uint_as_float(x[0]);
            v[4 + c] = __uint_as_float(x[1]);
          }
          store(row_of(i) + upper * 32 + l16, wn + (j + (quad & 1)) * 16 + (quad >> 1) * 8, v, 8);
        }
    }
  }
}

template <int OP, int DT, bool HIGH>
__global__ __launch_bounds__(HIGH ? 512 : 256, 2) void grouped_tile_kernel(const GroupedParams p) {
  __shared__ u32x4 smem[Shape<OP, DT, HIGH>::kLds / 16];
  tile_of<OP, DT, HIGH>(p, (int)blockIdx.x, smem, true);
}

// Both gradients: the weights' tiles fill the CUs that the rows' last round leaves idle.
template <int DT, bool HIGH>
__global__ __launch_bounds__(HIGH ? 512 : 256, 2) void grouped_tile_grads_kernel(const GroupedParams rows, const GroupedParams weights, const int first) {
  constexpr int kLds = Shape<kRowsGrad, DT, HIGH>::kLds, kLdsW = Shape<kWeightsGrad, DT, HIGH>::kLds;
  __shared__ u32x4 smem[(kLds > kLdsW ? kLds : kLdsW) / 16];
  if ((int)blockIdx.x < first) tile_of<kRowsGrad, DT, HIGH>(rows, (int)blockIdx.x, smem, false);
  else tile_of<kWeightsGrad, DT, HIGH>(weights, (int)blockIdx.x - first, smem, false);
}

// Blocks of a product, a multiple of eight.
long long blocks_of(const GroupedParams& p, int op, bool high, bool cut) {
  const int b = high ? 256 : 128;
  const long long tiles_n = ((op == kRows ? p.n : p.k) + b - 1) / b, tiles_w = ((long long)p.n + b - 1) / b * tiles_n;   // (of a weight)
  if (op == kWeightsGrad) return p.experts * ((tiles_w + 7) / 8) * 8;
  return (((p.rows / b + p.experts + 1) * tiles_n + 7) / 8 + (!cut ? 0 : high ? 24 : 32)) * 8;   // (parts of the last tiles)
}

}  // namespace

int grouped_tile_launch(const GroupedParams& p, int op, int dtype, bool high, hipStream_t stream) {
  const long long blocks = blocks_of(p, op, high, true);
  if (int rc = check_tiles(blocks, high ? 512 : 256)) return rc;
  const dim3 grid((unsigned)blocks), block(high ? 512 : 256);
#define CM_TILE(op_, dt)                                                                              \
  do {                                                                                                \
    if (high) hipLaunchKernelGGL((grouped_tile_kernel<op_, dt, true>), grid, block, 0, stream, p);    \
    else hipLaunchKernelGGL((grouped_tile_kernel<op_, dt, false>), grid, block, 0, stream, p);        \
  } while (0)
#define CM_TILE_OP(op_)                                              \
  do {                                                               \
    if (dtype == CPPMEGA_MI355_F16) CM_TILE(op_, CPPMEGA_MI355_F16); \
    else CM_TILE(op_, CPPMEGA_MI355_BF16);                           \
  } while (0)
  if (dtype == CPPMEGA_MI355_E4M3) CM_TILE(kRows, CPPMEGA_MI355_E4M3);
  else if (op == kRows) CM_TILE_OP(kRows);
  else if (op == kRowsGrad) CM_TILE_OP(kRowsGrad);
  else CM_TILE_OP(kWeightsGrad);
#undef CM_TILE_OP
#undef CM_TILE
  CM_HIP_CHECK(hipGetLastError());
  return 0;
}

int grouped_tile_grads_launch(const GroupedParams& rows, const GroupedParams& weights, int dtype, bool high, hipStream_t stream) {
  const long long first = blocks_of(rows, kRowsGrad, high, false), blocks = first + blocks_of(weights, kWeightsGrad, high, false);
  if (int rc = check_tiles(blocks, high ? 512 : 256)) return rc;
  const dim3 grid((unsigned)blocks), block(high ? 512 : 256);
#define CM_GRADS(dt)                                                                                                              \
  do {                                                                                                                            \
    if (high) hipLaunchKernelGGL((grouped_tile_grads_kernel<dt, true>), grid, block, 0, stream, rows, weights, (int)first);       \
    else hipLaunchKernelGGL((grouped_tile_grads_kernel<dt, false>), grid, block, 0, stream, rows, weights, (int)first);           \
  } while (0)
  if (dtype == CPPMEGA_MI355_F16) CM_GRADS(CPPMEGA_MI355_F16);
  else CM_GRADS(CPPMEGA_MI355_BF16);
#undef CM_GRADS
  CM_HIP_CHECK(hipGetLastError());
  return 0;
}

}  // namespace cm

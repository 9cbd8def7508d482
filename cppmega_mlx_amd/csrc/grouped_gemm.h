// What the kernels of the products grouped by expert share (gfx950).
//
// All three products are C = R Q^T summed over a contraction, tile by tile: R gives the rows of C, Q its columns (the axis
// that is contiguous in memory).
//                    rows of C (R)              columns of C (Q)         contraction
//   ROWS             tokens of e: x[t, :]       outputs: w[e, n, :]      k (contiguous in both)
//   ROWS_GRAD        tokens of e: dy[t, :]      inputs:  w[e, :, k]      n (contiguous in R, the slow axis of Q)
//   WEIGHTS_GRAD     outputs: dy[:, n]          inputs:  x[:, k]         tokens of e (the slow axis of both)
#pragma once

#include "common.h"
#include "gate.h"

namespace cm {

constexpr int kRows = CPPMEGA_MI355_GROUPED_ROWS, kRowsGrad = CPPMEGA_MI355_GROUPED_ROWS_GRAD, kWeightsGrad = CPPMEGA_MI355_GROUPED_WEIGHTS_GRAD;
constexpr int kMaxExperts = CPPMEGA_MI355_GROUPED_MAX_EXPERTS;

struct GroupedParams {
  const void *x, *w;
  void* y;
  const void* offsets;
  const float *x_scale, *w_scale;
  long long rows, x_pitch, w_pitch, y_pitch;
  int experts, n, k;
  int y_dtype, offsets64, x_scale_block, zero_tail;
  // the gated block: w is [experts, 2 n, k]; a tile's columns are as many of the gate's as of the up projection's
  int activation, pre_dtype;
  void* pre;
  long long pre_pitch;
};

typedef int i32x8 __attribute__((ext_vector_type(8)));

// Rows of expert e.  Offsets are what the device holds: they are brought into [0, rows], so that no kernel reads or writes outside.
__device__ __forceinline__ long long offset_of(const GroupedParams& p, int e) {
  if (!p.offsets) return e == 0 ? 0 : p.rows;                   // (one expert has all rows)
  const long long o = p.offsets64 ? ((const long long*)p.offsets)[e] : (long long)((const int*)p.offsets)[e];
  return o < 0 ? 0 : (o > p.rows ? p.rows : o);
}

// Row tiles of all experts in a row, BM rows each: the first tile of every expert in `starts` (kMaxExperts + 2 ints of LDS, filled by
// the first wavefront for the whole workgroup); their number comes back.  The rows behind the last expert are those of a last "expert"
// without a contraction when they are to be zeroed.  (Offsets that overlap may make more tiles than the launch has.)
template <int BM>
__device__ __forceinline__ int fill_tiles(const GroupedParams& p, int* starts) {
  if (threadIdx.x < 64) {
    const int lane = lane_id();
    int before = 0;
    const int entries = p.experts + 1;
    for (int e0 = 0; e0 < entries; e0 += 64) {
      const int e = e0 + lane;
      long long count = 0;
      if (e < entries) {
        const long long lo = offset_of(p, e), hi = e < p.experts ? offset_of(p, e + 1) : (p.zero_tail ? p.rows : lo);
        count = hi > lo ? hi - lo : 0;
      }
      const int tiles = (int)((count + BM - 1) / BM);
      const int through = (int)wave_inclusive_sum_dpp((unsigned)tiles);
      if (e < entries) starts[e] = before + through - tiles;
      before += __builtin_amdgcn_readlane(through, 63);
    }
    if (lane == 0) starts[entries] = before;
  }
  __syncthreads();
  const int total = starts[p.experts + 1], most = (int)(p.rows / BM) + p.experts + 1;
  return total < most ? total : most;
}
// the last entry whose first tile is <= t (entries without rows share their first tile with the next one)
__device__ __forceinline__ int expert_of_tile(const GroupedParams& p, const int* starts, int t) {
  int found = 0;
  for (int e0 = 0; e0 <= p.experts; e0 += 64) {
    const int e = e0 + lane_id();
    found += __popcll(__ballot(e <= p.experts && starts[e] <= t));
  }
  return __builtin_amdgcn_readfirstlane(found - 1);
}

// Tiles of BM rows of all experts in a row, found by every wavefront for itself (a scan over the counts in registers): which expert tile mt
// belongs to (p.experts: the rows behind them, to be zeroed), its first row and how many rows are there from it on.  false: no such tile.
template <int BM>
__device__ __forceinline__ bool rows_of_tile(const GroupedParams& p, int mt, int& e, int& first, int& rows) {
  const int lane = lane_id();
  e = -1; first = 0; rows = 0;
  for (int e0 = 0, before = 0; e0 <= p.experts; e0 += 64) {
    const int x = e0 + lane;
    int lo = 0, count = 0;
    if (x <= p.experts) {                                        // (the last entry: rows behind the experts)
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
      return true;
    }
    before = __builtin_amdgcn_readlane(through, 63);
  }
  return false;
}

// A launch has fewer than 2^32 threads.
inline int check_tiles(const char* call, long long tiles, int threads) {
  return tiles * threads > 0xffffffffll ? fail(CPPMEGA_MI355_ERR_UNSUPPORTED, "%s: %lld tiles in one call", call, tiles) : 0;
}

// Whether a kernel's launch has few enough tiles (asked before a call's first launch: one that is refused has written nothing), and the launch.
int grouped_general_check(const char* call, const GroupedParams& p, int op, bool gated);
int grouped_tile_check(const char* call, const GroupedParams& p, int op, bool high, bool gated);
int grouped_tile_grads_check(const char* call, const GroupedParams& rows, const GroupedParams& weights, bool high);
int grouped_stream_check(const char* call, const GroupedParams& p, bool gated);
int grouped_general_launch(const GroupedParams& p, int op, int dtype, bool gated, hipStream_t stream);
int grouped_tile_launch(const GroupedParams& p, int op, int dtype, bool high, bool gated, hipStream_t stream);
int grouped_tile_grads_launch(const GroupedParams& rows, const GroupedParams& weights, int dtype, bool high, hipStream_t stream);
int grouped_stream_launch(const GroupedParams& p, int dtype, bool gated, hipStream_t stream);

}  // namespace cm

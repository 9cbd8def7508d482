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
#include "mfma_util.h"

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
};

typedef int i32x8 __attribute__((ext_vector_type(8)));

// Rows of expert e.  Offsets are what the device holds: they are brought into [0, rows], so that no kernel reads or writes outside.
__device__ __forceinline__ long long offset_of(const GroupedParams& p, int e) {
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

// A launch has fewer than 2^32 threads.
inline int check_tiles(long long tiles, int threads) {
  return tiles * threads > 0xffffffffll ? fail(CPPMEGA_MI355_ERR_UNSUPPORTED, "grouped_gemm: %lld tiles in one call", tiles) : 0;
}

int grouped_general_launch(const GroupedParams& p, int op, int dtype, hipStream_t stream);
int grouped_tile_launch(const GroupedParams& p, int op, int dtype, bool high, hipStream_t stream);
int grouped_tile_grads_launch(const GroupedParams& rows, const GroupedParams& weights, int dtype, bool high, hipStream_t stream);
int grouped_stream_launch(const GroupedParams& p, int dtype, hipStream_t stream);

}  // namespace cm

// What the kernels of the products with 4-bit weights share (gfx950).
//
// Four bits become 16 + q in 16 bits by a shift and an and-or, two at a time: q lies where float16 and bfloat16 between 16 and 32 have their
// next four bits.  Products are exact; 16 times a group's sum of x comes off again in float32 with the bias,
//   y = sum over groups of s (sum x (16 + q)) + (b - 16 s) (sum x),
// the second part a product of its own with float32 operands, four groups to a matrix instruction.
// x is the first operand: a lane has one row of the weight in every sum, and with it one scale and one bias.
// A step is 128 channels, 16 bytes (32 codes) a lane; a word of it is eight channels, of which the low and the high half of a register
// take those four apart, so the pieces of x are put in that order.  With groups below 128 the four words of the four lanes of a row change
// places, so that one instruction has 32 channels in a run.
#pragma once

#include <type_traits>
#include <utility>

#include "grouped_gemm.h"

namespace cm {

struct W4Params {
  GroupedParams g;                                               // (w, scales: of 2 n rows when gated)
  const void *scale, *bias;
  int gated, log_split;                                          // wavefronts that divide the contraction
  int tile0;                                                     // the launch's first tile of rows
};

// Eight codes as 16 + q in 16 bits, in the order 0 4 1 5 2 6 3 7.
template <bool F16>
__device__ __forceinline__ bf16x8 widen(unsigned w, unsigned one) {        // (one: 16 twice, from a vector register, so that and-or is one instruction)
  constexpr unsigned mask = F16 ? 0x03c003c0u : 0x00780078u;
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

// A value of quad Q's lanes in the lanes of all quads (of the same place).
template <int Q>
__device__ __forceinline__ unsigned of_quad(unsigned v) {
  const u32x2 a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return __builtin_amdgcn_permlane16_swap(a[Q >> 1], a[Q >> 1], false, false)[Q & 1];
}

template <int N>
using Count = std::integral_constant<int, N>;
template <int... I, class F>
__device__ __forceinline__ void each(std::integer_sequence<int, I...>, F f) { (f(Count<I>()), ...); }
template <int N, class F>
__device__ __forceinline__ void each(F f) { each(std::make_integer_sequence<int, N>(), f); }

int w4_tile_launch(const W4Params& p, int group, bool f16, bool wide, hipStream_t stream);

}  // namespace cm

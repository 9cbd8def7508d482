// RMS norm of the residual stream and its gradients (gfx950).
//
//   h = round(x + residual),  s = 1 / sqrt(mean(h^2) + eps),  y = h s w        (y in the rows' type, or e4m3 with scales)
//   dx = dh + s g w - s^3 h mean(g w h),  dw = sum over rows of g h s          (g = dL/dy)
//
// Bound by memory: a row is read once into registers, reduced, and written from there.  A lane owns 8 consecutive channels of
// every THREADS * 8 (16-byte loads of 16-bit rows, at whatever alignment the row has), so that a 128-channel block of scales is
// 16 lanes.  Sums of squares, products with the weight, scales and the weight's gradient are float32; h is rounded once (it is
// the stream that the next layer reads, so y is the norm of what is stored), y once, from its float32 value, codes from float32 as well.
//
// Measured in a replayed graph, inputs in turn, bf16 with the residual: 8192 x 7168 82 us (5.7 TB/s; a large copy 4.9), e4m3 rows 74 us (5.6); 32768 x 1536
// 71 and 64; 1 x 7168 3.3 us, a launch.  Gradients: 8192 x 7168 75 us (6.3 TB/s), 4096 x 7168 41, 32768 x 1536 70.

#include "common.h"
#include "mfma_util.h"

namespace cm {
namespace {

constexpr int kF32 = CPPMEGA_MI355_F32, kF16 = CPPMEGA_MI355_F16;

// 8 consecutive channels as they lie in memory
template <int DT>
struct Raw {
  u32x4 q[DT == kF32 ? 2 : 1];
};
template <int DT>
struct Elem { typedef unsigned short type; };
template <>
struct Elem<kF32> { typedef float type; };

template <int DT>
__device__ __forceinline__ Raw<DT> load8(const typename Elem<DT>::type* p, int valid) {
  Raw<DT> r;
  if (valid >= 8) {
    __builtin_memcpy(&r, p, sizeof(r));
  } else {
    typename Elem<DT>::type e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = i < valid ? p[i] : 0;
    __builtin_memcpy(&r, e, sizeof(r));
  }
  return r;
}
template <int DT>
__device__ __forceinline__ void store8(typename Elem<DT>::type* p, const Raw<DT>& r, int valid) {
  if (valid >= 8) {
    __builtin_memcpy(p, &r, sizeof(r));
  } else {
    typename Elem<DT>::type e[8];
    __builtin_memcpy(e, &r, sizeof(r));
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < valid) p[i] = e[i];
  }
}
template <int DT>
__device__ __forceinline__ void unpack8(const Raw<DT>& r, float (&v)[8]) {
  if constexpr (DT == kF32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r.q[i >> 2][i & 3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned w = r.q[0][i >> 1];
      if constexpr (DT == kF16) v[i] = f16_bits_to_f32((unsigned short)((i & 1) ? w >> 16 : w & 0xffffu));
      else v[i] = __uint_as_float((i & 1) ? w & 0xffff0000u : w << 16);
    }
  }
}
template <int DT>
__device__ __forceinline__ Raw<DT> pack8(const float (&v)[8]) {
  Raw<DT> r;
  if constexpr (DT == kF32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.q[i >> 2][i & 3] = __float_as_uint(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) r.q[0][i] = DT == kF16 ? pack_f16(v[2 * i], v[2 * i + 1]) : pack_bf16(v[2 * i], v[2 * i + 1]);
  }
  return r;
}

// ---- reductions: vector instructions only --------------------------------------------------
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xf, 0xf, true));
}
template <bool MAX>
__device__ __forceinline__ float both(float a, float b) { return MAX ? fmaxf(a, b) : a + b; }
// over the lane's group of 16, which every lane gets: partners 1 and 2 apart, then the mirrored quad and half
template <bool MAX>
__device__ __forceinline__ float over16(float v) {
  v = both<MAX>(v, dpp<0xB1>(v));
  v = both<MAX>(v, dpp<0x4E>(v));
  v = both<MAX>(v, dpp<0x141>(v));
  return both<MAX>(v, dpp<0x140>(v));
}
template <bool MAX>
__device__ __forceinline__ float over_wave(float v) {
  v = over16<MAX>(v);
  v = both<MAX>(v, xor16(v));
  return both<MAX>(v, xor32(v));
}
// over the THREADS threads that share a row; `slots` holds a float per wavefront and is free again behind the next barrier
template <bool MAX, int THREADS>
__device__ __forceinline__ float over_row(float v, float* slots) {
  v = over_wave<MAX>(v);
  if constexpr (THREADS > 64) {
    constexpr int W = THREADS / 64;
    if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = v;
    __syncthreads();
    v = slots[0];
#pragma unroll
    for (int i = 1; i < W; ++i) v = both<MAX>(v, slots[i]);
  }
  return v;
}

// v / 448: the product with 1 / 448, corrected by its remainder (infinities have none)
__device__ __forceinline__ float over448(float v) {
  const float q = v * (1.0f / 448.0f);
  return v < __builtin_inff() ? fmaf(fmaf(-448.0f, q, v), 1.0f / 448.0f, q) : q;
}
// The exponent of the smallest power of two s with 448 s >= amax: amax = fr * 2^ex, fr in [0.5, 1), and 448 = 0.875 * 2^9.  float32 has none below
// 2^-149; no power reaches an infinite amax, whose scale is infinite like the other kind's.  0 for zeros and NaN.
__device__ __forceinline__ int exponent_of(float amax) {
  if (!(amax > 0.0f)) return 0;
  if (!(amax < __builtin_inff())) return 1024;
  int ex;
  const float fr = frexpf(amax, &ex);
  ex += fr > 0.875f ? -8 : -9;
  return ex < -149 ? -149 : ex;
}

// v / s for r = 1 / s, to the last bit but for rare ties of the quotient: the remainder corrects the product.  An infinite
// scale keeps the plain product (0, or NaN for infinities), whose remainder would be NaN.
__device__ __forceinline__ float quotient(float v, float s, float r) {
  const float q = v * r;
  const float c = fmaf(fmaf(-q, s, v), r, q);
  return s < __builtin_inff() ? c : q;
}
__device__ __forceinline__ unsigned codes4(float a, float b, float c, float d) {
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
}

struct NormParams {
  const void *x, *residual, *weight;
  void *out, *residual_out;
  float* scale;
  long long first, rows, x_pitch, residual_pitch, out_pitch, residual_out_pitch;   // (a launch has rows first .. rows - 1)
  int width, scale_block, pow2;
  float eps;
};

// THREADS threads to a row (64: four rows to a workgroup), PER pieces of 8 channels to a thread.
template <int DT, bool WF32, bool FP8, int THREADS, int PER>
__global__ __launch_bounds__(THREADS == 64 ? 256 : THREADS) void rms_norm_kernel(const NormParams p) {
  typedef typename Elem<DT>::type T;
  constexpr int WT = WF32 ? kF32 : DT;
  __shared__ float slots[2][16];
  const int tid = THREADS == 64 ? (int)(threadIdx.x & 63) : (int)threadIdx.x;
  const long long row = p.first + (THREADS == 64 ? (long long)blockIdx.x * 4 + (threadIdx.x >> 6) : (long long)blockIdx.x);
  if (THREADS == 64 && row >= p.rows) return;
  const T* x = (const T*)p.x + row * p.x_pitch;
  float v[PER][8];
  Raw<WT> w[PER];
  {
    Raw<DT> xr[PER], rr[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = (i * THREADS + tid) * 8;
      xr[i] = load8<DT>(x + c, p.width - c);
    }
    if (p.residual) {
      const T* r = (const T*)p.residual + row * p.residual_pitch;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int c = (i * THREADS + tid) * 8;
        rr[i] = load8<DT>(r + c, p.width - c);
      }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = (i * THREADS + tid) * 8;
      w[i] = load8<WT>((const typename Elem<WT>::type*)p.weight + c, p.width - c);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      unpack8<DT>(xr[i], v[i]);
      if (p.residual) {
        float r[8];
        unpack8<DT>(rr[i], r);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] += r[e];
        const Raw<DT> h = pack8<DT>(v[i]);
        unpack8<DT>(h, v[i]);
        const int c = (i * THREADS + tid) * 8;
        if (p.residual_out) store8<DT>((T*)p.residual_out + row * p.residual_out_pitch + c, h, p.width - c);
      }
    }
  }
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < PER; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf(v[i][e], v[i][e], sum);
  sum = over_row<false, THREADS>(sum, slots[0]);
  const float s = 1.0f / sqrtf(sum / (float)p.width + p.eps);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    float wv[8];
    unpack8<WT>(w[i], wv);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[i][e] = FP8 ? v[i][e] * wv[e] : v[i][e] * s * wv[e];
  }
  if constexpr (!FP8) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = (i * THREADS + tid) * 8;
      store8<DT>((T*)p.out + row * p.out_pitch + c, pack8<DT>(v[i]), p.width - c);
    }
  } else {
    float am[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      am[i] = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) am[i] = fmaxf(am[i], fabsf(v[i][e]));
    }
    if (!p.scale_block) {
#pragma unroll
      for (int i = 1; i < PER; ++i) am[0] = fmaxf(am[0], am[i]);
      am[0] = over_row<true, THREADS>(am[0], slots[1]);
    }
    const int blocks = (p.width + 127) / 128;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = (i * THREADS + tid) * 8, valid = p.width - c;
      // y / scale = h w s / (max |h w| s / 448) = 448 h w / max |h w|: without s and the roundings that come with it, and for bf16, whose products and
      // their 448 times are exact, with one rounding in all, so that a tie stays one (8192 x 7168 bf16 rows: every code is that of 64 bits; 159 of 59
      // million are not with the largest over 448 as the divisor, 4000 with y / scale).  A scale that is rounded to a power of two or held at its least divides y itself.
      const float top = p.scale_block ? over16<true>(am[i]) : am[0];
      float q[8], sc;
      if (p.pow2) {
        // (by the exponent: the reciprocal of a scale of 2^-128 or less is no float32)
        const int ex = exponent_of(top * s);
        sc = ldexpf(1.0f, ex);
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] = ldexpf(v[i][e] * s, -ex);
      } else {
        sc = fmaxf(over448(top * s), 1.0e-12f);
        const bool cancels = sc > 1.0e-12f && top < 0x1p119f;    // (448 h w is finite)
        const float d = cancels ? top : sc, r = 1.0f / d, f = cancels ? 448.0f : s;
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] = quotient(v[i][e] * f, d, r);
      }
      const uint2 codes = make_uint2(codes4(q[0], q[1], q[2], q[3]), codes4(q[4], q[5], q[6], q[7]));
      unsigned char* const to = (unsigned char*)p.out + row * p.out_pitch + c;
      if (valid >= 8) {
        __builtin_memcpy(to, &codes, 8);
      } else {
        for (int e = 0; e < 8; ++e)
          if (e < valid) to[e] = (unsigned char)((e < 4 ? codes.x : codes.y) >> (8 * (e & 3)));
      }
      if (p.scale_block) {
        if ((tid & 15) == 0 && valid > 0) p.scale[row * blocks + (c >> 7)] = sc;
      } else if (tid == 0 && i == 0) {
        p.scale[row] = sc;
      }
    }
  }
}

// ---- gradients -----------------------------------------------------------------------------
struct NormBwdParams {
  const void *dy, *h, *weight, *dh;
  void* dx;
  float *dweight, *partial;
  long long rows, dy_pitch, h_pitch, dh_pitch, dx_pitch;
  int width, groups;
  float eps;
};

// Group g of THREADS threads takes rows g, g + groups, ..; its sums for the weight stay in registers until its last row and go
// to partial[g].  TWICE: rows too wide for the registers of 1024 threads beside those sums are read again (from the caches) for
// their second use.  Above 16384 channels a thread's sums of 32 channels do not fit all the same (48 to 252 bytes a lane go to memory):
// 2048 x 32768 bf16 139 us (2.9 TB/s), float32 383; of 16384 channels 44 and 104.
template <int DT, bool WF32, int THREADS, int PER, bool TWICE>
__global__ __launch_bounds__(THREADS == 64 ? 256 : THREADS) void rms_norm_bwd_kernel(const NormBwdParams p) {
  typedef typename Elem<DT>::type T;
  constexpr int WT = WF32 ? kF32 : DT, W = THREADS / 64;
  __shared__ float slots[2][2][16];
  const int tid = THREADS == 64 ? (int)(threadIdx.x & 63) : (int)threadIdx.x;
  const int group = THREADS == 64 ? (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6) : (int)blockIdx.x;
  if (THREADS == 64 && group >= p.groups) return;
  constexpr int KEPT = TWICE ? 1 : PER;
  Raw<WT> w[KEPT];
  float dw[PER][8];
  const typename Elem<WT>::type* const weight = (const typename Elem<WT>::type*)p.weight;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int c = (i * THREADS + tid) * 8;
    if (!TWICE) w[i] = load8<WT>(weight + c, p.width - c);
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[i][e] = 0.0f;
  }
  int turn = 0;
  for (long long row = group; row < p.rows; row += p.groups, turn ^= 1) {
    Raw<DT> g[KEPT], h[KEPT], d[KEPT];
    const T* const dy = (const T*)p.dy + row * p.dy_pitch;
    const T* const hrow = (const T*)p.h + row * p.h_pitch;
    const T* const dh = (const T*)p.dh + row * p.dh_pitch;
    if (!TWICE) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int c = (i * THREADS + tid) * 8;
        h[i] = load8<DT>(hrow + c, p.width - c);
        g[i] = load8<DT>(dy + c, p.width - c);
      }
      if (p.dh) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int c = (i * THREADS + tid) * 8;
          d[i] = load8<DT>(dh + c, p.width - c);
        }
      }
    }
    float squares = 0.0f, cross = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = TWICE ? 0 : i, c = (i * THREADS + tid) * 8;
      if (TWICE) {
        h[0] = load8<DT>(hrow + c, p.width - c);
        g[0] = load8<DT>(dy + c, p.width - c);
        w[0] = load8<WT>(weight + c, p.width - c);
      }
      float gv[8], hv[8], wv[8];
      unpack8<DT>(g[at], gv);
      unpack8<DT>(h[at], hv);
      unpack8<WT>(w[at], wv);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        squares = fmaf(hv[e], hv[e], squares);
        cross = fmaf(gv[e] * wv[e], hv[e], cross);
      }
      if (TWICE) __builtin_amdgcn_sched_barrier(0);     // (one piece at a time: all of them ahead do not fit)
    }
    squares = over_wave<false>(squares);
    cross = over_wave<false>(cross);
    if constexpr (THREADS > 64) {
      // (two sets of slots in turn: a row's are read behind its barrier, the next row's are others)
      if ((threadIdx.x & 63) == 0) {
        slots[turn][0][threadIdx.x >> 6] = squares;
        slots[turn][1][threadIdx.x >> 6] = cross;
      }
      __syncthreads();
      squares = slots[turn][0][0];
      cross = slots[turn][1][0];
#pragma unroll
      for (int k = 1; k < W; ++k) {
        squares += slots[turn][0][k];
        cross += slots[turn][1][k];
      }
    }
    const float s = 1.0f / sqrtf(squares / (float)p.width + p.eps);
    const float c3 = cross / (float)p.width * s * s * s;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = TWICE ? 0 : i, c = (i * THREADS + tid) * 8;
      if (TWICE) {
        h[0] = load8<DT>(hrow + c, p.width - c);
        g[0] = load8<DT>(dy + c, p.width - c);
        w[0] = load8<WT>(weight + c, p.width - c);
        if (p.dh) d[0] = load8<DT>(dh + c, p.width - c);
      }
      float gv[8], hv[8], wv[8], dv[8];
      unpack8<DT>(g[at], gv);
      unpack8<DT>(h[at], hv);
      unpack8<WT>(w[at], wv);
      if (p.dh) unpack8<DT>(d[at], dv);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        dw[i][e] = fmaf(gv[e] * s, hv[e], dw[i][e]);
        const float dx = fmaf(gv[e] * wv[e], s, -c3 * hv[e]);
        gv[e] = p.dh ? dx + dv[e] : dx;
      }
      store8<DT>((T*)p.dx + row * p.dx_pitch + c, pack8<DT>(gv), p.width - c);
      if (TWICE) __builtin_amdgcn_sched_barrier(0);
    }
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int c = (i * THREADS + tid) * 8;
    store8<kF32>(p.partial + (size_t)group * p.width + c, pack8<kF32>(dw[i]), p.width - c);
  }
}

// dweight[c] = the partial sums of column c, group by group in 16 runs that are added in order
__global__ __launch_bounds__(1024) void rms_norm_dweight_kernel(const float* partial, float* dweight, int groups, int width) {
  __shared__ float runs[16][64];
  const int lane = lane_id(), run = (int)(threadIdx.x >> 6), c = (int)blockIdx.x * 64 + lane;
  float sum = 0.0f;
  if (c < width) {
    // (eight loads on their way at a time: one after the other, 512 groups took 11 us)
    int g = run;
    for (; g + 7 * 16 < groups; g += 8 * 16) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = partial[(size_t)(g + 16 * i) * width + c];
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += v[i];
    }
    for (; g < groups; g += 16) sum += partial[(size_t)g * width + c];
  }
  runs[run][lane] = sum;
  __syncthreads();
  if (run == 0 && c < width) {
#pragma unroll
    for (int i = 1; i < 16; ++i) sum += runs[i][lane];
    dweight[c] = sum;
  }
}

// Groups of the gradient kernel: four rows each, so that their partial sums (float32, written and read) stay below the rows' traffic, but
// 256 at least (a workgroup for every CU; of rows of up to 1024 channels, four groups to a workgroup, for a quarter of them: 1024 x 1024 bf16
// take 10 us, 4096 x 1024 14), and at most 1024 threads of them to a CU (512 of narrow rows).  Measured, us with 256 / 512 / 1024 groups:
// 512 x 7168 14 / 17 / 17, 2048 x 4096 22 / 18 / 21, 8192 x 4096 61 / 44 / 42, 4096 x 7168 50 / 41 / 48, 2048 x 16384 54 / 59 / 71.
int bwd_groups(long long rows, int width) {
  const long long most = width <= 1024 ? 2048 : width <= 4096 ? 1024 : width <= 8192 ? 512 : 256;
  const long long groups = rows / 4 < 256 ? 256 : rows / 4 < most ? rows / 4 : most;
  return (int)(rows < groups ? rows : groups);
}

// Rows of up to 1024 channels: one wavefront, without a barrier (32768 x 1024 42 us, e4m3 39; 256 threads 50 and 58; of 2048 channels 93 and 84; 92 and 81).
// Of up to 8192: a thread for every 8 channels where rows are few and latency counts (7168 channels, us of 1 / 512 rows: 3.2 / 7.2,
// with 512 threads 3.5 / 7.7), half as many where they are not (4096 rows, e4m3: 37, with 1024 threads 39).  A launch has fewer than 2^32 threads.
template <int DT, bool WF32, bool FP8>
void launch_norm(NormParams p, hipStream_t stream) {
  const long long total = p.rows, most = 1 << 21;
  for (p.first = 0; p.first < total; p.first += most) {
    p.rows = total - p.first < most ? total : p.first + most;
    const unsigned rows = (unsigned)(p.rows - p.first);
#define CM_NORM(threads, per) \
  hipLaunchKernelGGL((rms_norm_kernel<DT, WF32, FP8, threads, per>), dim3(threads == 64 ? (rows + 3) / 4 : rows), dim3(threads == 64 ? 256 : threads), 0, stream, p)
    if (p.width <= 512) CM_NORM(64, 1);
    else if (p.width <= 1024) CM_NORM(64, 2);
    else if (p.width <= 2048) CM_NORM(256, 1);
    else if (p.width <= 4096) CM_NORM(256, 2);
    else if (p.width <= 8192 && total > 512) CM_NORM(512, 2);
    else if (p.width <= 8192) CM_NORM(1024, 1);
    else if (p.width <= 16384) CM_NORM(1024, 2);
    else CM_NORM(1024, 4);
#undef CM_NORM
  }
}

template <int DT, bool WF32>
void launch_bwd(const NormBwdParams& p, hipStream_t stream) {
  const unsigned groups = (unsigned)p.groups;
#define CM_BWD(threads, per) \
  hipLaunchKernelGGL((rms_norm_bwd_kernel<DT, WF32, threads, per, (threads == 1024 && per > 1)>), dim3(threads == 64 ? (groups + 3) / 4 : groups), dim3(threads == 64 ? 256 : threads), 0, stream, p)
  if (p.width <= 512) CM_BWD(64, 1);
  else if (p.width <= 1024) CM_BWD(64, 2);
  else if (p.width <= 2048) CM_BWD(256, 1);
  else if (p.width <= 4096) CM_BWD(256, 2);
  else if (p.width <= 8192) CM_BWD(512, 2);
  else if (p.width <= 16384) CM_BWD(1024, 2);
  else CM_BWD(1024, 4);
#undef CM_BWD
}

bool float_type(int dt) { return dt == CPPMEGA_MI355_F32 || dt == CPPMEGA_MI355_F16 || dt == CPPMEGA_MI355_BF16; }

int check_bwd(const cppmega_mi355_rms_norm_bwd_args_t& a) {
  if (a.rows < 0 || a.rows > 0x7fffffffll || a.width < 1 || a.width > CPPMEGA_MI355_NORM_MAX_WIDTH)
    return fail(CPPMEGA_MI355_ERR_SHAPE, "rms_norm_bwd: rows=%lld width=%d (width must be in [1, %d])", (long long)a.rows, a.width, CPPMEGA_MI355_NORM_MAX_WIDTH);
  if (!float_type(a.dtype) || (a.weight_dtype != CPPMEGA_MI355_F32 && a.weight_dtype != a.dtype))
    return fail(CPPMEGA_MI355_ERR_DTYPE, "rms_norm_bwd: rows of dtype %d with a weight of dtype %d", a.dtype, a.weight_dtype);
  return 0;
}

}  // namespace

int rms_norm_launch(const cppmega_mi355_rms_norm_args_t& a, hipStream_t stream) {
  if (a.rows < 0 || a.rows > 0x7fffffffll || a.width < 1 || a.width > CPPMEGA_MI355_NORM_MAX_WIDTH)
    return fail(CPPMEGA_MI355_ERR_SHAPE, "rms_norm: rows=%lld width=%d (width must be in [1, %d])", (long long)a.rows, a.width, CPPMEGA_MI355_NORM_MAX_WIDTH);
  if (!float_type(a.x_dtype) || (a.weight_dtype != CPPMEGA_MI355_F32 && a.weight_dtype != a.x_dtype))
    return fail(CPPMEGA_MI355_ERR_DTYPE, "rms_norm: rows of dtype %d with a weight of dtype %d", a.x_dtype, a.weight_dtype);
  const bool fp8 = a.out_dtype == CPPMEGA_MI355_E4M3;
  if (!fp8 && a.out_dtype != a.x_dtype) return fail(CPPMEGA_MI355_ERR_DTYPE, "rms_norm: out must have the rows' type or be e4m3, got dtype %d", a.out_dtype);
  if (fp8 && a.scale_block != 0 && a.scale_block != 128)
    return fail(CPPMEGA_MI355_ERR_SHAPE, "rms_norm: scale_block must be 0 (per row) or 128, got %d", a.scale_block);
  if (!(a.eps >= 0.0f) || a.eps > 3.0e38f) return fail(CPPMEGA_MI355_ERR_SHAPE, "rms_norm: eps must be finite and not negative");
  if (a.rows == 0) return 0;
  if (!a.x || !a.weight || !a.out || (fp8 && !a.scale)) return fail(CPPMEGA_MI355_ERR_NULL, "rms_norm: x / weight / out / scale is NULL");
  if (a.residual_out && !a.residual) return fail(CPPMEGA_MI355_ERR_NULL, "rms_norm: residual_out without a residual");
  NormParams p;
  p.x = a.x; p.residual = a.residual; p.weight = a.weight; p.out = a.out; p.residual_out = a.residual_out; p.scale = a.scale;
  p.rows = a.rows; p.x_pitch = a.x_pitch; p.residual_pitch = a.residual_pitch; p.out_pitch = a.out_pitch; p.residual_out_pitch = a.residual_out_pitch;
  p.width = a.width; p.scale_block = a.scale_block; p.pow2 = a.pow2_scales; p.eps = a.eps;
  const bool wf32 = a.weight_dtype == CPPMEGA_MI355_F32;
#define CM_TYPE(dt, wf)                                 \
  do {                                                  \
    if (fp8) launch_norm<dt, wf, true>(p, stream);      \
    else launch_norm<dt, wf, false>(p, stream);         \
  } while (0)
  if (a.x_dtype == CPPMEGA_MI355_F32) CM_TYPE(CPPMEGA_MI355_F32, true);
  else if (a.x_dtype == CPPMEGA_MI355_F16 && wf32) CM_TYPE(CPPMEGA_MI355_F16, true);
  else if (a.x_dtype == CPPMEGA_MI355_F16) CM_TYPE(CPPMEGA_MI355_F16, false);
  else if (wf32) CM_TYPE(CPPMEGA_MI355_BF16, true);
  else CM_TYPE(CPPMEGA_MI355_BF16, false);
#undef CM_TYPE
  CM_HIP_CHECK(hipGetLastError());
  return 0;
}

int rms_norm_bwd_workspace_bytes(const cppmega_mi355_rms_norm_bwd_args_t& a, size_t* bytes) {
  const int rc = check_bwd(a);
  if (rc) return rc;
  *bytes = (size_t)bwd_groups(a.rows, a.width) * (size_t)a.width * sizeof(float);
  return 0;
}

int rms_norm_bwd_launch(const cppmega_mi355_rms_norm_bwd_args_t& a, hipStream_t stream) {
  const int rc = check_bwd(a);
  if (rc) return rc;
  if (!(a.eps >= 0.0f) || a.eps > 3.0e38f) return fail(CPPMEGA_MI355_ERR_SHAPE, "rms_norm_bwd: eps must be finite and not negative");
  if (!a.dweight || (a.rows > 0 && (!a.dy || !a.h || !a.weight || !a.dx)))
    return fail(CPPMEGA_MI355_ERR_NULL, "rms_norm_bwd: dy / h / weight / dx / dweight is NULL");
  NormBwdParams p;
  p.dy = a.dy; p.h = a.h; p.weight = a.weight; p.dh = a.dh; p.dx = a.dx; p.dweight = a.dweight; p.partial = (float*)a.workspace;
  p.rows = a.rows; p.dy_pitch = a.dy_pitch; p.h_pitch = a.h_pitch; p.dh_pitch = a.dh_pitch; p.dx_pitch = a.dx_pitch;
  p.width = a.width; p.groups = bwd_groups(a.rows, a.width); p.eps = a.eps;
  const size_t need = (size_t)p.groups * (size_t)p.width * sizeof(float);
  if (need && (!a.workspace || a.workspace_bytes < need))
    return fail(CPPMEGA_MI355_ERR_WORKSPACE, "rms_norm_bwd: workspace of %zu bytes needed, %zu given", need, a.workspace ? a.workspace_bytes : (size_t)0);
  if (p.groups) {
    const bool wf32 = a.weight_dtype == CPPMEGA_MI355_F32;
    if (a.dtype == CPPMEGA_MI355_F32) launch_bwd<CPPMEGA_MI355_F32, true>(p, stream);
    else if (a.dtype == CPPMEGA_MI355_F16 && wf32) launch_bwd<CPPMEGA_MI355_F16, true>(p, stream);
    else if (a.dtype == CPPMEGA_MI355_F16) launch_bwd<CPPMEGA_MI355_F16, false>(p, stream);
    else if (wf32) launch_bwd<CPPMEGA_MI355_BF16, true>(p, stream);
    else launch_bwd<CPPMEGA_MI355_BF16, false>(p, stream);
    CM_HIP_CHECK(hipGetLastError());
  }
  hipLaunchKernelGGL(rms_norm_dweight_kernel, dim3((unsigned)(p.width + 63) / 64), dim3(1024), 0, stream, (const float*)p.partial, p.dweight, p.groups, p.width);
  CM_HIP_CHECK(hipGetLastError());
  return 0;
}

}  // namespace cm

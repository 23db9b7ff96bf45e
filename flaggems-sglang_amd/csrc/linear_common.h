// Shared by the 16-bit products (linear.hip, linear_small.hip): parameters,
// element types, the groups of rows, activations.
#pragma once

#include <algorithm>
#include <atomic>
#include <string>

#include "dense_common.h"
#include "gemm_tiled_common.h"

namespace fgs {

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

template <int TY>
struct Mma16;
template <>
struct Mma16<FGS_DTYPE_BF16> {
  typedef bf16x8 Frag;
  static __device__ __forceinline__ f32x16 mma32(Frag a, Frag b, f32x16 c) {
    return mfma32_bf16(a, b, c);
  }
  static __device__ __forceinline__ f32x4 mma16(Frag a, Frag b, f32x4 c) {
    return mfma16_bf16(a, b, c);
  }
};
template <>
struct Mma16<FGS_DTYPE_FP16> {
  typedef f16x8 Frag;
  static __device__ __forceinline__ f32x16 mma32(Frag a, Frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mma16(Frag a, Frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

// Four rows of 16 values in LDS, a row to 16 lanes, column by column: lane i of 16
// gives the address of four values of row i / 4, from column 4 (i % 4) on, and has
// the four of column i. (__restrict__: with no scope of its own the compiler takes
// the read for one of the bytes that the loads in flight will write, and waits for
// all of those first.)
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* LdsWords;
__device__ __forceinline__ s16x4 read_transposed(LdsWords __restrict__ at) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(at);
}

// ---------------------------------------------------------- groups of rows ---
// Rows come sorted by group: group e has counts[e] of them, from row 0 on.
// Counts are the device's: a negative one counts as 0, and those that pass the
// last row are cut, so every row named below exists. A wave handles 64 groups a
// step; every lane returns the same values.
struct GroupScan {
  const int32_t* counts;
  int groups, rows;

  // Inclusive sums over the lanes that stay at `rows` (at most 2^30) once there.
  __device__ __forceinline__ int sums(int v) const {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(v, d, 64);
      if (lane >= d) v = min(v + o, rows);
    }
    return v;
  }
  __device__ __forceinline__ int count(int e) const {
    return e < groups ? min(max(counts[e], 0), rows) : 0;
  }

  // First row and rows of group e.
  __device__ __forceinline__ void range(int e, int* first, int* n) const {
    int base = 0;
    for (int e0 = 0;; e0 += 64) {
      const int incl = min(base + sums(count(e0 + (threadIdx.x & 63))), rows);
      if (e < e0 + 64) {
        const int end = __builtin_amdgcn_readlane(incl, e - e0);
        const int start = e > e0 ? __builtin_amdgcn_readlane(incl, e - e0 - 1) : base;
        *first = start;
        *n = end - start;
        return;
      }
      base = __builtin_amdgcn_readlane(incl, 63);
    }
  }
  // Tiles of bm rows that the groups and the rows behind them (the group
  // `groups`) need, none over two groups.
  __device__ __forceinline__ int tiles(int bm) const {
    int base = 0, total = 0;
    for (int e0 = 0; e0 < groups; e0 += 64) {
      const int c = count(e0 + (threadIdx.x & 63));
      const int s = sums(c), lane = threadIdx.x & 63;
      const int end = min(base + s, rows);
      const int prev = __shfl_up(end, 1, 64);
      const int start = lane ? prev : base;
      int t = (end - start + bm - 1) / bm;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) t += __shfl_xor(t, d, 64);
      total += __builtin_amdgcn_readfirstlane(t);
      base = __builtin_amdgcn_readlane(end, 63);
    }
    return total + (rows - base + bm - 1) / bm;
  }
  // Tile t: its group, first row and rows.
  __device__ __forceinline__ void tile(int t, int bm, int* e, int* first, int* n) const {
    int base = 0;
    const int lane = threadIdx.x & 63;
    for (int e0 = 0; e0 < groups; e0 += 64) {
      const int end = min(base + sums(count(e0 + lane)), rows);
      const int prev = __shfl_up(end, 1, 64);
      const int start = lane ? prev : base;
      const int own = (end - start + bm - 1) / bm;
      int incl = own;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(incl, d, 64);
        if (lane >= d) incl += o;
      }
      const uint64_t hit = __ballot(incl > t);
      if (hit) {
        const int l = __ffsll(static_cast<long long>(hit)) - 1;
        const int at = t - __builtin_amdgcn_readlane(incl - own, l);
        const int s = __builtin_amdgcn_readlane(start, l);
        *e = e0 + l;
        *first = s + at * bm;
        *n = min(bm, __builtin_amdgcn_readlane(end, l) - *first);
        return;
      }
      t -= __builtin_amdgcn_readlane(incl, 63);
      base = __builtin_amdgcn_readlane(end, 63);
    }
    *e = groups;
    *first = base + t * bm;
    *n = min(bm, rows - *first);
  }
};

// Two values of a 16-bit type in a word.
template <int TY>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (TY == FGS_DTYPE_BF16) return cvt_pk_bf16(lo, hi);
  return Elem<TY>::from_f32(lo) | static_cast<uint32_t>(Elem<TY>::from_f32(hi)) << 16;
}

// ------------------------------------------------------------- activations ---
// erfc(x) / exp(-x^2) for x >= 0 as t times a polynomial in t = 1 / (1 + x / 2),
// fitted to scaled erfc at Chebyshev nodes over x in [0, 10.5] (least squares of
// the relative error, 5e-8 there; 3.3e-7 with fp32's steps): the normal
// distribution's tail with its leading digits, which 1 + erf loses, and without a
// branch. Behind 10.5 exp(-x^2) vanishes in fp32.
__device__ __forceinline__ float scaled_erfc(float x) {
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.5f, x, 1.f));
  float p = -0.060205210000276566f;
  p = __builtin_fmaf(p, t, 0.28990432620048523f);
  p = __builtin_fmaf(p, t, -0.497749924659729f);
  p = __builtin_fmaf(p, t, 0.28953269124031067f);
  p = __builtin_fmaf(p, t, -0.03407368063926697f);
  p = __builtin_fmaf(p, t, 0.2056339681148529f);
  p = __builtin_fmaf(p, t, 0.24241343140602112f);
  p = __builtin_fmaf(p, t, 0.2824624478816986f);
  p = __builtin_fmaf(p, t, 0.2820819020271301f);
  return p * t;
}
// Phi(-|z|) of the normal distribution, and exp(-z^2 / 2).
__device__ __forceinline__ float normal_tail(float z, float* e) {
  *e = __expf(-0.5f * z * z);
  return 0.5f * *e * scaled_erfc(0.70710678118654752f * fabsf(z));
}

template <int ACT>
__device__ __forceinline__ float linear_act(float z) {
  if constexpr (ACT == FGS_ACT_SILU) return z * __builtin_amdgcn_rcpf(1.f + __expf(-z));
  if constexpr (ACT == FGS_ACT_GELU) {
    float e;
    const float tail = normal_tail(z, &e);
    return z * (z < 0.f ? tail : 1.f - tail);
  }
  if constexpr (ACT == FGS_ACT_RELU) return z < 0.f ? 0.f : z;
  return z;
}
// act(z) and its derivative there.
template <int ACT>
__device__ __forceinline__ float linear_act_slope(float z, float* slope) {
  if constexpr (ACT == FGS_ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + __expf(-z));
    *slope = s * __builtin_fmaf(z, 1.f - s, 1.f);
    return z * s;
  }
  if constexpr (ACT == FGS_ACT_GELU) {
    float e;
    const float tail = normal_tail(z, &e);
    const float phi = z < 0.f ? tail : 1.f - tail;
    *slope = __builtin_fmaf(z, 0.39894228040143268f * e, phi);
    return z * phi;
  }
  if constexpr (ACT == FGS_ACT_RELU) {
    *slope = z <= 0.f ? 0.f : 1.f;  // (1 of a NaN)
    return z < 0.f ? 0.f : z;
  }
  *slope = 1.f;
  return z;
}

// f(std::integral_constant<int, ACT>) for a runtime activation.
template <class F>
int with_act(int act, F&& f) {
  switch (act) {
    case FGS_ACT_RELU: return f(std::integral_constant<int, FGS_ACT_RELU>{});
    case FGS_ACT_SILU: return f(std::integral_constant<int, FGS_ACT_SILU>{});
    case FGS_ACT_GELU: return f(std::integral_constant<int, FGS_ACT_GELU>{});
    default: return f(std::integral_constant<int, FGS_ACT_NONE>{});
  }
}

// f(std::integral_constant<int, i>) for i = 0 .. N - 1 (a loop that is surely
// unrolled: registers cannot be indexed).
template <int N, int I = 0, class F>
__device__ __forceinline__ void static_for(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    static_for<N, I + 1>(f);
  }
}

// ---------------------------------------------------------------- launches ---
int launch_linear_small(const LinearParams& p, int mode, int dtype, int form, hipStream_t stream);

// Tiles of bm rows for any division of the rows into the groups and what lies behind
// them, each of which may end in a tile of its own.
inline int64_t linear_row_tiles(const LinearParams& p, int bm) {
  const int64_t rows = p.rows, whole = (rows + bm - 1) / bm;
  return p.counts ? std::min(rows, whole + p.groups) : whole;
}

// Operands whose sums run across their rows: a stage's resource ends with the last
// row's last column, and the next row has to begin behind that.
inline int check_linear_across(const LinearParams& p, int mode) {
  if ((mode == kLinearWgrad && p.ldq < p.m) ||
      ((mode == kLinearWgrad || mode == kLinearDgrad) && p.ldp < p.n))
    return fail(FGS_EUNSUPPORTED, "rows that overlap: their stride is less than their width");
  return FGS_OK;
}

// Launches `kernel` with more than 64 KiB of LDS, which each GPU has to be told
// of once (`told`: a bit a GPU).
template <class... P, class... A>
inline int launch_lds(const char* name, void (*kernel)(P...), std::atomic<uint64_t>& told, int64_t wgs,
               int threads, int lds, hipStream_t stream, A... args) {
  if (wgs * threads > 0xffffffffll) return fail(FGS_EUNSUPPORTED, "too many tiles for a grid");
  int gpu = 0;
  hipError_t e = hipGetDevice(&gpu);
  const uint64_t bit = uint64_t{1} << (gpu & 63);
  if (e == hipSuccess && (gpu > 63 || !(told.load(std::memory_order_relaxed) & bit))) {
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                            hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e == hipSuccess && gpu <= 63) told.fetch_or(bit, std::memory_order_relaxed);
  }
  if (e != hipSuccess) return fail(FGS_ELAUNCH, std::string(name) + ": " + hipGetErrorString(e));
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(wgs)), dim3(threads), lds, stream, args...);
  return check_launch(name);
}

}  // namespace fgs

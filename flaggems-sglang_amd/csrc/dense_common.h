// Shared pieces of the dense operators around the routed experts (norm_quant.hip,
// block_gemm.hip): element types, 8-value vectors, and the 8-bit codes of
// values held in fp32.
#pragma once

#include "fgs_moe_kernels.h"

namespace fgs {

// ---------------------------------------------------------- element types ---
template <int TY>
struct Elem;
template <>
struct Elem<FGS_DTYPE_BF16> {
  typedef uint16_t raw;
  static __device__ __forceinline__ float to_f32(raw v) { return bf16_bits_to_f32(v); }
  static __device__ __forceinline__ raw from_f32(float v) { return f32_to_bf16_bits(v); }
};
template <>
struct Elem<FGS_DTYPE_FP16> {
  typedef uint16_t raw;
  static __device__ __forceinline__ float to_f32(raw v) {
    return static_cast<float>(__builtin_bit_cast(_Float16, v));
  }
  static __device__ __forceinline__ raw from_f32(float v) {
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
  }
};
template <>
struct Elem<FGS_DTYPE_FP32> {
  typedef float raw;
  static __device__ __forceinline__ float to_f32(raw v) { return v; }
  static __device__ __forceinline__ raw from_f32(float v) { return v; }
};

// Eight consecutive values as they lie in memory. VEC: the address is 16-byte
// aligned and all eight exist (one or two 16-byte loads); otherwise the first
// `valid` (any more count as 8) are read one by one and the others are 0.
template <int TY, bool VEC>
struct Vec8 {
  typedef typename Elem<TY>::raw raw;
  static constexpr int N = sizeof(raw) / 2;  // 16-byte words
  u32x4 w[N];

  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = u32x4{0, 0, 0, 0};
  }
  __device__ __forceinline__ void load(const void* base, int64_t at, int64_t valid) {
    const raw* p = static_cast<const raw*>(base) + at;
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const u32x4*>(p)[i];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const raw v = j < valid ? p[j] : raw{0};
        if constexpr (N == 2) w[j / 4][j % 4] = __float_as_uint(v);
        else if (j & 1) w[0][j / 2] |= static_cast<uint32_t>(v) << 16;
        else w[0][j / 2] = v;
      }
    }
  }
  __device__ __forceinline__ float operator[](int j) const {
    if constexpr (N == 2) return __uint_as_float(w[j / 4][j % 4]);
    else if constexpr (TY == FGS_DTYPE_BF16)
      return __uint_as_float((j & 1) ? w[0][j / 2] & 0xffff0000u : w[0][j / 2] << 16);
    else
      return Elem<TY>::to_f32(
          static_cast<raw>((j & 1) ? w[0][j / 2] >> 16 : w[0][j / 2] & 0xffffu));
  }
};

template <int TY, bool VEC>
__device__ __forceinline__ void store8(void* base, int64_t at, int64_t valid, const float (&f)[8]) {
  typedef typename Elem<TY>::raw raw;
  raw* p = static_cast<raw*>(base) + at;
  if constexpr (VEC) {
    constexpr int N = sizeof(raw) / 2;
    u32x4 w[N];
#pragma unroll
    for (int i = 0; i < 4 * N; ++i) {
      uint32_t u;
      if constexpr (N == 2) u = __float_as_uint(f[i]);
      else if constexpr (TY == FGS_DTYPE_BF16) u = cvt_pk_bf16(f[2 * i], f[2 * i + 1]);
      else u = Elem<TY>::from_f32(f[2 * i]) |
               static_cast<uint32_t>(Elem<TY>::from_f32(f[2 * i + 1])) << 16;
      w[i / 4][i % 4] = u;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) reinterpret_cast<u32x4*>(p)[i] = w[i];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < valid) p[j] = Elem<TY>::from_f32(f[j]);
  }
}

// ------------------------------------------------------------ lane moves ---
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t x) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, 0xF, 0xF, false));
}
template <int CTRL>
__device__ __forceinline__ float dpp_f32(float x) {
  return __uint_as_float(dpp_u32<CTRL>(__float_as_uint(x)));
}

// Largest of the 16 lanes of a row / of the wave's 64, and the wave's sum, in
// every lane: quad permutations and row mirrors, then the four rows' lanes.
// The whole wave calls.
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  v = max(v, dpp_u32<0xB1>(v));   // quad_perm [1, 0, 3, 2]
  v = max(v, dpp_u32<0x4E>(v));   // quad_perm [2, 3, 0, 1]
  v = max(v, dpp_u32<0x141>(v));  // row_half_mirror
  return max(v, dpp_u32<0x140>(v));  // row_mirror
}
__device__ __forceinline__ uint32_t lane_u32(uint32_t v, int lane) {
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
  v = row_max(v);
  return max(max(lane_u32(v, 0), lane_u32(v, 16)), max(lane_u32(v, 32), lane_u32(v, 48)));
}
__device__ __forceinline__ float wave_sum_f32(float v) {
  v += dpp_f32<0xB1>(v);
  v += dpp_f32<0x4E>(v);
  v += dpp_f32<0x141>(v);
  v += dpp_f32<0x140>(v);
  const uint32_t b = __float_as_uint(v);
  return (__uint_as_float(lane_u32(b, 0)) + __uint_as_float(lane_u32(b, 16))) +
         (__uint_as_float(lane_u32(b, 32)) + __uint_as_float(lane_u32(b, 48)));
}

// -------------------------------------------------------------- 8-bit codes ---
// |f| as an integer whose order is that of the magnitudes, a NaN above all:
// a NaN in a group is the group's largest value, so its scale is NaN.
__device__ __forceinline__ uint32_t abs_bits(float f) { return __float_as_uint(f) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t abs_bits8(const float (&f)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, abs_bits(f[j]));
  return m;
}
// max(amax, 1e-10) / top, NaN where the largest is one.
__device__ __forceinline__ float scale_of(uint32_t amax, float top) {
  return __uint_as_float(max(amax, __float_as_uint(1e-10f))) / top;
}

// Eight values over their scale as codes. |f| / scale is at most the format's
// largest value times 1 + 2^-23 (scale is a rounded quotient and at least
// 1e-10 / 448), which rounds to that value: neither format needs a clamp. A
// NaN scale (a NaN in the group) gives e4m3 NaN codes and int8 zeros, an
// infinite one zeros, and NaN / zero for the infinity itself.
__device__ __forceinline__ uint2 codes_fp8(const float (&f)[8], float scale) {
  const float inv = 1.0f / scale, res = residual_scale(scale);
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    w[i] = cvt_pk_fp8(quotient(f[4 * i], res, inv), quotient(f[4 * i + 1], res, inv)) |
           cvt_pk_fp8(quotient(f[4 * i + 2], res, inv), quotient(f[4 * i + 3], res, inv)) << 16;
  return uint2{w[0], w[1]};
}
__device__ __forceinline__ uint2 codes_int8(const float (&f)[8], float scale) {
  const float inv = 1.0f / scale, res = residual_scale(scale);
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float t = __builtin_rintf(quotient(f[j], res, inv));
    const int32_t c = t == t ? static_cast<int32_t>(t) : 0;
    w[j / 4] |= (static_cast<uint32_t>(c) & 0xffu) << (8 * (j & 3));
  }
  return uint2{w[0], w[1]};
}
template <bool VEC>
__device__ __forceinline__ void store_codes(uint8_t* p, int64_t valid, uint2 c) {
  if constexpr (VEC) {
    *reinterpret_cast<uint2*>(p) = c;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < valid) p[j] = static_cast<uint8_t>((j < 4 ? c.x : c.y) >> (8 * (j & 3)));
  }
}

}  // namespace fgs

// Row operators around the dense 8-bit products: the root-mean-square norm
// with the residual's addition and an output in 16 / 32 and / or 8 bits, and
// the gated activation with an output in 8 bits.
//
// Both hold a row's values in registers in fp32 (8 consecutive ones a vector,
// NV vectors a thread), so every input is read once whatever the outputs are:
// they are bound by memory, or by one load-reduce-store latency where rows
// are few. A 128-column group of the e4m3 scales is 16 neighbouring lanes, so
// its largest value is four DPP moves.
#include <algorithm>
#include <string>

#include "dense_common.h"

namespace fgs {

constexpr int kRowThreads = 1024;   // most threads a row gets
constexpr int kRowVecs = 8;         // most vectors a thread holds
static_assert(kRowMaxCols == 8 * kRowThreads * kRowVecs, "columns a workgroup holds");

// Sum / maximum over the workgroup's waves (`red` has a word a wave).
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = wave_sum_f32(v);
  const int nw = blockDim.x / 64;
  if (nw == 1) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
  for (int i = 0; i < nw; ++i) s += red[i];
  return s;
}
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* red) {
  v = wave_max_u32(v);
  const int nw = blockDim.x / 64;
  if (nw == 1) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  uint32_t s = 0;
  for (int i = 0; i < nw; ++i) s = max(s, red[i]);
  return s;
}

// ------------------------------------------------------------------- norm ---
// h = x + residual; n = h / sqrt(mean(h^2) + eps) * (weight + offset), all in
// fp32: the residual output is h rounded once, the norm output n rounded once,
// and the 8-bit codes and scales come from the unrounded n.
// WAVE: a wave takes a row (4 a workgroup), else the workgroup one row.
// Bound by memory with many rows: bf16 with residual and all four outputs, 8192
// x 7168, 97 us (5.5 TB/s); by load, sum and store one after the other with few:
// 1 x 7168 3.5 us, 61 x 4096 without codes 2.7. Column-major scales leave as
// single words, each a 32-byte sector of its own: 309 MB written where row-major
// ones take 295, 97 us and 95 (the product that reads them gains more: its loads).
// Rows of odd length one value a load: 4096 x 7168 45 us, x 7167 163.
template <int TY, int WTY, bool VEC, bool WAVE, bool RES, int NV>
__global__ __launch_bounds__(WAVE ? 256 : kRowThreads) void rms_norm_kernel(
    const RmsNormParams p) {
  __shared__ float red_sum[kRowThreads / 64];
  __shared__ uint32_t red_max[kRowThreads / 64];
  const int tid = WAVE ? threadIdx.x & 63 : threadIdx.x;
  const int threads = WAVE ? 64 : blockDim.x;
  const int64_t row = WAVE ? blockIdx.x * int64_t{4} + (threadIdx.x >> 6) : blockIdx.x;
  if (WAVE && row >= p.rows) return;
  auto col = [&](int v) { return (static_cast<int64_t>(v) * threads + tid) * 8; };

  // Every load of the row first, the weight's among them; rows of more than
  // two vectors a thread in batches and the weight later, to stay in registers.
  constexpr int BATCH = NV <= 2 ? NV : sizeof(typename Elem<TY>::raw) == 2 && NV == 4 ? 4 : 2;
  constexpr bool EARLY = NV <= 2;
  Vec8<WTY, VEC> w[EARLY ? NV : 1];
  float h[NV][8];
  float sum = 0.f;
#pragma unroll
  for (int v0 = 0; v0 < NV; v0 += BATCH) {
    Vec8<TY, VEC> x[BATCH], r[RES ? BATCH : 1];
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const int64_t c = col(v0 + b);
      x[b].zero();
      if constexpr (EARLY) w[b].zero();
      if constexpr (RES) r[b].zero();
      if (c < p.cols) {
        x[b].load(p.x, row * p.x_stride + c, p.cols - c);
        if constexpr (RES) r[b].load(p.residual, row * p.res_stride + c, p.cols - c);
        if constexpr (EARLY) w[b].load(p.weight, c, p.cols - c);
      }
    }
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const int v = v0 + b;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        h[v][j] = x[b][j];
        if constexpr (RES) h[v][j] += r[b][j];
        sum = __builtin_fmaf(h[v][j], h[v][j], sum);
      }
      if constexpr (RES) {
        const int64_t c = col(v);
        if (c < p.cols) store8<TY, VEC>(p.res_out, row * p.res_out_stride + c, p.cols - c, h[v]);
      }
    }
  }
  sum = WAVE ? wave_sum_f32(sum) : block_sum(sum, red_sum);
  const float rstd = 1.0f / sqrtf(sum / static_cast<float>(p.cols) + p.eps);

  uint32_t amax = 0;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int64_t c = col(v);
    if constexpr (!EARLY) {
      w[0].zero();
      if (c < p.cols) w[0].load(p.weight, c, p.cols - c);
    }
    const Vec8<WTY, VEC>& wv = w[EARLY ? v : 0];
    // columns past the row: 0, whatever rstd is
#pragma unroll
    for (int j = 0; j < 8; ++j)
      h[v][j] = c + (VEC ? 0 : j) < p.cols ? h[v][j] * rstd * (wv[j] + p.offset) : 0.f;
    if (p.norm && c < p.cols) store8<TY, VEC>(p.norm, row * p.cols + c, p.cols - c, h[v]);
    if (p.quant == FGS_QUANT_FP8_GROUP) {
      const float scale = scale_of(row_max(abs_bits8(h[v])), 448.f);
      if (c < p.cols) {
        store_codes<VEC>(p.q + row * p.cols + c, p.cols - c, codes_fp8(h[v], scale));
        if ((tid & 15) == 0) p.scales[row * p.s_row + (c >> 7) * p.s_col] = scale;
      }
    } else if (p.quant == FGS_QUANT_INT8_TOKEN) {
      amax = max(amax, abs_bits8(h[v]));
    }
  }
  if (p.quant != FGS_QUANT_INT8_TOKEN) return;
  amax = WAVE ? wave_max_u32(amax) : block_max(amax, red_max);
  const float scale = scale_of(amax, 127.f);
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int64_t c = (static_cast<int64_t>(v) * threads + tid) * 8;
    if (c < p.cols)
      store_codes<VEC>(p.q + row * p.cols + c, p.cols - c, codes_int8(h[v], scale));
  }
  if (tid == 0) p.scales[row * p.s_row] = scale;
}

// ------------------------------------------------------- gated activation ---
// v = act(gate) * up in fp32 (gate the row's first n columns, up the other n),
// quantised unrounded. e4m3: a workgroup takes blockDim * NV * 8 columns of a
// row (grid y); int8, whose scale is the row's: the whole row.
// The exact gelu by erfc, which keeps its relative accuracy for negative gates
// (1 + erf cancels there), and the silu with the rounding of its exponent's
// argument made good: a scale may come from such values alone.
// bf16 to e4m3, 8192 x 14336 115 us (5.1 TB/s), 8 x 2048 2.1 us, with gelu 190
// and 2.7 (erfc's instructions). Column-major scales are a 32-byte sector each:
// 147 MB written, 121 with row-major ones, 114 us and 111. 4096 x 7168 30 us, x
// 7167 71.
__device__ __forceinline__ float gelu_tail_mul(float g, float u) {
  return 0.5f * g * erfcf(-0.70710678118654752f * g) * u;
}

// o = silu(g) * u = g / (1 + exp(-g)) * u of eight values, within 8 u (u = 2^-24).
// exp(-g) = 2^t (1 - w) with t = fl(-g / ln 2) and w = t ln 2 + g, what the
// rounding of t left (ln 2 in two floats); with 2^t alone the result is |g| u
// off: 58 u at -87.
// REFINED: the quotient by a residual step instead of a product with the
// reciprocal. An int8 code is a whole step off where a value lies on the wrong
// side of a tie: of 40 x 2.6 million codes 3 differ from those of the formula
// in rounded steps, 13 without it. 999 x 2560 to int8 5.95 us, 5.75 without, 5.5
// with 2^t alone; e4m3, whose steps do not show it: 8192 x 14336 121, 117, 114.
// A vector with a gate beyond 87 takes the plain formula, and below -87, where
// exp(-g) overflows, g exp(g) u in halves: so a gate of +infinity gives
// infinity, and one of -infinity NaN (infinity times zero).
template <bool REFINED>
__device__ __forceinline__ void silu_mul8(const float (&g)[8], const float (&u)[8],
                                          float (&o)[8]) {
  float far = 0.f;  // (a NaN is not: both ways give NaN)
#pragma unroll
  for (int j = 0; j < 8; ++j) far = fmaxf(far, fabsf(g[j]));
  if (far <= 87.f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float t = -1.44269504088896341f * g[j];
      const float w = __builtin_fmaf(t, -1.90465429995776e-9f,
                                     __builtin_fmaf(t, 0.693147182464599609375f, g[j]));
      const float e = __builtin_amdgcn_exp2f(t);
      const float d = 1.0f + __builtin_fmaf(-w, e, e), r = __builtin_amdgcn_rcpf(d);
      float q = g[j] * r;
      if constexpr (REFINED) q = __builtin_fmaf(__builtin_fmaf(-d, q, g[j]), r, q);
      o[j] = q * u[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float half = expf(0.5f * g[j]);
      o[j] = g[j] < -87.f ? (g[j] * half) * (half * u[j]) : g[j] / (1.0f + expf(-g[j])) * u[j];
    }
  }
}

template <int TY, bool VEC, bool WAVE, int NV>
__global__ __launch_bounds__(WAVE ? 256 : kRowThreads) void gated_quant_kernel(
    const GatedQuantParams p) {
  __shared__ uint32_t red_max[kRowThreads / 64];
  const int tid = WAVE ? threadIdx.x & 63 : threadIdx.x;
  const int threads = WAVE ? 64 : blockDim.x;
  const int64_t row = WAVE ? blockIdx.x * int64_t{4} + (threadIdx.x >> 6) : blockIdx.x;
  if (WAVE && row >= p.rows) return;
  const int64_t first = static_cast<int64_t>(blockIdx.y) * threads * NV;

  // vectors loaded at once
  constexpr int BATCH = NV <= 2 ? NV : NV == 8 && TY == FGS_DTYPE_FP32 ? 1 : 2;
  float h[NV][8];
  uint32_t amax = 0;
#pragma unroll
  for (int v0 = 0; v0 < NV; v0 += BATCH) {
    Vec8<TY, VEC> g[BATCH], u[BATCH];
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const int64_t c = (first + static_cast<int64_t>(v0 + b) * threads + tid) * 8;
      g[b].zero();
      u[b].zero();
      if (c < p.n) {
        g[b].load(p.x, row * p.x_stride + c, p.n - c);
        u[b].load(p.x, row * p.x_stride + p.n + c, p.n - c);
      }
    }
    if (p.act == kActGelu) {
#pragma unroll
      for (int b = 0; b < BATCH; ++b)
#pragma unroll
        for (int j = 0; j < 8; ++j) h[v0 + b][j] = gelu_tail_mul(g[b][j], u[b][j]);
    } else {
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        float gate[8], up[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          gate[j] = g[b][j];
          up[j] = u[b][j];
        }
        if (p.quant == FGS_QUANT_INT8_TOKEN) silu_mul8<true>(gate, up, h[v0 + b]);
        else silu_mul8<false>(gate, up, h[v0 + b]);
      }
    }
  }
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int64_t c = (first + static_cast<int64_t>(v) * threads + tid) * 8;
    if (p.quant == FGS_QUANT_FP8_GROUP) {
      const float scale = scale_of(row_max(abs_bits8(h[v])), 448.f);
      if (c < p.n) {
        store_codes<VEC>(p.q + row * p.n + c, p.n - c, codes_fp8(h[v], scale));
        if ((tid & 15) == 0) p.scales[row * p.s_row + (c >> 7) * p.s_col] = scale;
      }
    } else {
      amax = max(amax, abs_bits8(h[v]));
    }
  }
  if (p.quant == FGS_QUANT_FP8_GROUP) return;
  amax = WAVE ? wave_max_u32(amax) : block_max(amax, red_max);
  const float scale = scale_of(amax, 127.f);
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int64_t c = (static_cast<int64_t>(v) * threads + tid) * 8;
    if (c < p.n) store_codes<VEC>(p.q + row * p.n + c, p.n - c, codes_int8(h[v], scale));
  }
  if (tid == 0) p.scales[row * p.s_row] = scale;
}

// -------------------------------------------------------------- launchers ---
namespace {

// Vectors a thread holds and threads of a row of `chunks` vectors: `wave`
// for a wave a row.
struct RowShape {
  bool wave;
  int nv, threads;
};
// Few rows leave CUs idle, so a row takes as many threads as it has vectors;
// with many, threads hold two vectors (more loads in flight for the same waves:
// norm with e4m3 output, 4096 x 7168: 34.8 us, 40.7 with one, 39.6 with four;
// 1021 x 3584 to int8 8.0, 8.6, 8.4), and rows of at most 64 vectors take a wave
// each, four a workgroup (norm with e4m3 output, 4096 x 128: 3.7 us, 4.1 with a
// workgroup each; two and four vectors a lane lost against workgroups: 4096 x
// 1024 8.8 / 8.2, 4096 x 2048 15.6 / 13.3).
RowShape row_shape(int64_t rows, int64_t chunks, bool vec) {
  if (vec && rows >= 1024 && chunks <= 64) return {true, 1, 256};
  int nv = 1;
  while (nv < kRowVecs && chunks > int64_t{kRowThreads} * nv) nv *= 2;
  if (rows >= 512 && nv < 4 && chunks >= 128 * nv) nv *= 2;
  const int64_t t = (chunks + nv - 1) / nv;
  return {false, nv, static_cast<int>((t + 63) / 64 * 64)};
}

template <class F>
int with_nv(int nv, F&& f) {
  switch (nv) {
    case 1: return f(std::integral_constant<int, 1>{});
    case 2: return f(std::integral_constant<int, 2>{});
    case 4: return f(std::integral_constant<int, 4>{});
    default: return f(std::integral_constant<int, 8>{});
  }
}
template <class F>
int with_type(int ty, F&& f) {
  switch (ty) {
    case FGS_DTYPE_BF16: return f(std::integral_constant<int, FGS_DTYPE_BF16>{});
    case FGS_DTYPE_FP16: return f(std::integral_constant<int, FGS_DTYPE_FP16>{});
    default: return f(std::integral_constant<int, FGS_DTYPE_FP32>{});
  }
}

// The runtime counts a grid in 32-bit threads.
int check_grid(const dim3& grid, int threads) {
  if (static_cast<int64_t>(grid.x) * threads > 0xffffffffll)
    return fail(FGS_EUNSUPPORTED, "too many rows for a grid");
  return FGS_OK;
}
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
int64_t elem_bytes(int ty) { return ty == FGS_DTYPE_FP32 ? 4 : 2; }

}  // namespace

int launch_rms_norm(const RmsNormParams& p, int dtype, int weight_dtype, hipStream_t stream) {
  if (p.rows == 0) return FGS_OK;
  const int64_t es = elem_bytes(dtype);
  const bool vec = p.cols % 8 == 0 && aligned16(p.x) && aligned16(p.weight) && aligned16(p.norm) &&
                   p.x_stride * es % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(p.q) % 8 == 0 &&
                   (!p.residual || (aligned16(p.residual) && aligned16(p.res_out) &&
                                    p.res_stride * es % 16 == 0 &&
                                    p.res_out_stride * es % 16 == 0));
  const RowShape s = row_shape(p.rows, (p.cols + 7) / 8, vec);
  const dim3 grid(static_cast<unsigned>(s.wave ? (p.rows + 3) / 4 : p.rows));
  if (const int rc = check_grid(grid, s.threads)) return rc;
  const int rc = with_type(dtype, [&](auto ty) {
    constexpr int TY = decltype(ty)::value;
    auto go = [&](auto wty) {
      constexpr int WTY = decltype(wty)::value;
      auto run = [&](auto res) {
        constexpr bool RES = decltype(res)::value;
        return with_nv(s.nv, [&](auto nv) {
          constexpr int NV = decltype(nv)::value;
          auto kernel = vec ? rms_norm_kernel<TY, WTY, true, false, RES, NV>
                            : rms_norm_kernel<TY, WTY, false, false, RES, NV>;
          if constexpr (NV == 1) {
            if (s.wave) kernel = rms_norm_kernel<TY, WTY, true, true, RES, NV>;
          }
          hipLaunchKernelGGL(kernel, grid, dim3(s.threads), 0, stream, p);
          return FGS_OK;
        });
      };
      return p.residual ? run(std::true_type{}) : run(std::false_type{});
    };
    if (weight_dtype == FGS_DTYPE_FP32) return go(std::integral_constant<int, FGS_DTYPE_FP32>{});
    return go(ty);
  });
  return rc ? rc : check_launch("rms_norm_kernel");
}

int launch_gated_quant(const GatedQuantParams& p, int dtype, hipStream_t stream) {
  if (p.rows == 0) return FGS_OK;
  const bool vec = p.n % 8 == 0 && aligned16(p.x) && p.x_stride * elem_bytes(dtype) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(p.q) % 8 == 0;
  const int64_t chunks = (p.n + 7) / 8;
  RowShape s = row_shape(p.rows, chunks, vec);
  unsigned gy = 1;
  // e4m3 groups are apart, so a row takes several workgroups of 256 threads --
  // but for wide rows of more than the 256 MB cache beside the memory holds,
  // which read their two halves best as a whole (bf16 by parts and whole: 2048 x
  // 14336 31 and 35 us, 4096 57 and 61, 6000 87 and 84, 8192 118 and 111, 16384
  // 238 and 213; 8192 x 7168 56 and 54, 52 and 53 where the input was just used;
  // 32768 x 7168 240 and 205, 16384 x 4096 61 and 61).
  const bool whole = p.n >= 6144 && p.rows * p.n * 2 * elem_bytes(dtype) > int64_t{256} << 20;
  if (p.quant == FGS_QUANT_FP8_GROUP && !s.wave && !whole) {
    s.nv = 1;
    s.threads = static_cast<int>(std::min<int64_t>(256, (chunks + 63) / 64 * 64));
    gy = static_cast<unsigned>((chunks + s.threads - 1) / s.threads);
  }
  const dim3 grid(static_cast<unsigned>(s.wave ? (p.rows + 3) / 4 : p.rows), gy);
  if (const int rc = check_grid(grid, s.threads)) return rc;
  const int rc = with_type(dtype, [&](auto ty) {
    constexpr int TY = decltype(ty)::value;
    return with_nv(s.nv, [&](auto nv) {
      constexpr int NV = decltype(nv)::value;
      auto kernel =
          vec ? gated_quant_kernel<TY, true, false, NV> : gated_quant_kernel<TY, false, false, NV>;
      if constexpr (NV == 1) {
        if (s.wave) kernel = gated_quant_kernel<TY, true, true, NV>;
      }
      hipLaunchKernelGGL(kernel, grid, dim3(s.threads), 0, stream, p);
      return FGS_OK;
    });
  });
  return rc ? rc : check_launch("gated_quant_kernel");
}

}  // namespace fgs

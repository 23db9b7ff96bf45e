// Tokens sorted by expert and back.
//
// The order is the alignment's (align.hip) with blocks of one row: expert by
// expert, within one by slot, the slots that no expert here has behind them. All
// kernels go token by token, so that a token's row is read (or written) once and
// its slots' rows in between; a thread has one vector of 16 bytes of a row, so
// that a token's row is spread over as many lanes as it has vectors. Rows of at
// least 16 bytes go in whole vectors at any alignment: a row's last vector ends
// with the row and overlaps the one before (the same values twice). Bound by the
// slots' rows.
#include <algorithm>

#include "dense_common.h"

namespace fgs {

// ---------------------------------------------------------------- vectors ---
// Sixteen bytes (or one value, for rows shorter than that) at any address.
template <int TY, bool WHOLE>
struct RowVec {
  typedef typename Elem<TY>::raw raw;
  static constexpr int N = WHOLE ? 16 / sizeof(raw) : 1;
  raw v[N];
  __device__ __forceinline__ void load(const void* p) { __builtin_memcpy(v, p, sizeof(v)); }
  __device__ __forceinline__ void store(void* p) const { __builtin_memcpy(p, v, sizeof(v)); }
  __device__ __forceinline__ float operator[](int j) const { return Elem<TY>::to_f32(v[j]); }
  __device__ __forceinline__ void set(int j, float f) { v[j] = Elem<TY>::from_f32(f); }
};

// Vectors of a row of n values, N each, and where vector i starts.
__device__ __host__ __forceinline__ int64_t row_vectors(int64_t n, int N) {
  return (n + N - 1) / N;
}
__device__ __forceinline__ int64_t vector_at(int64_t i, int64_t n, int N) {
  return i * N + N <= n ? i * N : n - N;
}

// Threads a token takes: a power of two, at most a workgroup.
static int token_lanes_log2(int64_t vectors) {
  int l = 0;
  while (l < 8 && (int64_t{1} << l) < vectors) ++l;
  return l;
}

constexpr int kAtOnce = 8;  // slots whose rows a thread has in flight

// ---------------------------------------------------------- tokens -> rows ---
// rows[row of (t, k)] = x[t] (as bytes). With the ids, the row of a slot that no
// expert here has is one behind all experts' and gets zeros, and the order's final
// form is written; without, such a slot has no row (-1), and the workgroups behind
// the tokens' clear the rows that have no slot.
template <int W>
__global__ __launch_bounds__(256) void permute_kernel(const PermuteParams p, int lanes_log2,
                                                      int token_wgs) {
  struct Word {
    uint8_t b[W];
  };
  const int lanes = 1 << lanes_log2;
  if (static_cast<int>(blockIdx.x) >= token_wgs) {
    const int64_t row = (blockIdx.x - token_wgs) * int64_t{256 >> lanes_log2} +
                        (threadIdx.x >> lanes_log2);
    if (row >= p.m * p.topk || p.slot_of_row[row] >= 0) return;
    const int64_t i = (threadIdx.x & (lanes - 1)) + blockIdx.y * int64_t{lanes};
    if (i >= row_vectors(p.bytes, W)) return;
    const Word zero{};
    __builtin_memcpy(p.rows + row * p.bytes + vector_at(i, p.bytes, W), &zero, W);
    return;
  }
  const int64_t t = blockIdx.x * int64_t{256 >> lanes_log2} + (threadIdx.x >> lanes_log2);
  if (t >= p.m) return;
  const int64_t i = (threadIdx.x & (lanes - 1)) + blockIdx.y * int64_t{lanes};
  if (i >= row_vectors(p.bytes, W)) return;
  const int64_t at = vector_at(i, p.bytes, W);
  Word v;
  __builtin_memcpy(&v, p.x + t * p.x_stride + at, W);
  for (int k0 = 0; k0 < p.topk; k0 += kAtOnce) {
    int row[kAtOnce], id[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int64_t s = t * p.topk + min(k0 + j, p.topk - 1);
      row[j] = p.ids ? p.place[s] : p.row_of_slot[s];
      id[j] = p.ids ? p.ids[s] : 0;
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      if (k0 + j >= p.topk) break;
      const bool kept = p.ids ? id[j] >= 0 && id[j] < p.experts
                              : row[j] >= 0 && row[j] < p.m * p.topk;
      if (p.ids && i == 0) {
        const int64_t s = t * p.topk + k0 + j;
        p.row_of_slot[s] = kept ? row[j] : -1;
        p.slot_of_row[row[j]] = kept ? static_cast<int32_t>(s) : -1;
      }
      if (!kept && !p.ids) continue;
      Word o = v;
      if (!kept) o = Word{};
      __builtin_memcpy(p.rows + row[j] * p.bytes + at, &o, W);
    }
  }
}

template <int W>
static int permute_width(const PermuteParams& p, hipStream_t stream) {
  const int64_t vecs = row_vectors(p.bytes, W);
  const int l = token_lanes_log2(vecs);
  const int64_t per = 256 >> l;
  const int64_t tokens = (p.m + per - 1) / per;
  const int64_t tail = p.ids ? 0 : (p.m * p.topk + per - 1) / per;
  const int64_t chunks = (vecs + (int64_t{1} << l) - 1) >> l;
  if (tokens + tail > 0xffffffll || chunks > 0xffff)
    return fail(FGS_EUNSUPPORTED, "too many rows or columns for a grid");
  hipLaunchKernelGGL(permute_kernel<W>,
                     dim3(static_cast<unsigned>(tokens + tail), static_cast<unsigned>(chunks)),
                     dim3(256), 0, stream, p, l, static_cast<int>(tokens));
  return check_launch("permute_kernel");
}
int launch_permute(const PermuteParams& p, hipStream_t stream) {
  if (p.bytes >= 16) return permute_width<16>(p, stream);
  if (p.bytes >= 4) return permute_width<4>(p, stream);
  return permute_width<1>(p, stream);
}

// ---------------------------------------------------------- rows -> tokens ---
// out[t] = sum_k w[t, k] rows[row of (t, k)], in fp32 from k = 0 on; a slot
// without a row (outside [0, n_rows)) adds nothing, whatever its weight is.
template <int TY, bool WHOLE, bool WEIGHTS>
__global__ __launch_bounds__(256) void unpermute_kernel(const UnpermuteParams p, int lanes_log2) {
  typedef RowVec<TY, WHOLE> V;
  typedef typename V::raw raw;
  const int lanes = 1 << lanes_log2;
  const int64_t t = blockIdx.x * int64_t{256 >> lanes_log2} + (threadIdx.x >> lanes_log2);
  if (t >= p.m) return;
  const int64_t i = (threadIdx.x & (lanes - 1)) + blockIdx.y * int64_t{lanes};
  if (i >= row_vectors(p.cols, V::N)) return;
  const int64_t at = vector_at(i, p.cols, V::N);
  const raw* rows = static_cast<const raw*>(p.rows);
  float acc[V::N] = {};
  for (int k0 = 0; k0 < p.topk; k0 += kAtOnce) {
    int row[kAtOnce];
    float w[kAtOnce];
    V v[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int64_t s = t * p.topk + min(k0 + j, p.topk - 1);
      row[j] = k0 + j < p.topk ? p.row_of_slot[s] : -1;
      if constexpr (WEIGHTS) w[j] = p.weights[s];
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j)
      if (row[j] >= 0 && row[j] < p.n_rows) v[j].load(rows + row[j] * p.ld + at);
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j)
      if (row[j] >= 0 && row[j] < p.n_rows)
#pragma unroll
        for (int c = 0; c < V::N; ++c)
          acc[c] = WEIGHTS ? __builtin_fmaf(w[j], v[j][c], acc[c]) : acc[c] + v[j][c];
  }
  V o;
#pragma unroll
  for (int c = 0; c < V::N; ++c) o.set(c, acc[c]);
  o.store(static_cast<raw*>(p.out) + t * p.cols + at);
}

// The gradients: drows[row of (t, k)] = w[t, k] dout[t] (rows without a slot: 0),
// dweights[t, k] = <dout[t], rows[row of (t, k)]>, 0 without a row. `waves` waves
// have a token; a row's dot product is added up lane by lane, over the lanes and
// over the waves, always in the same order.
template <int TY, bool WHOLE>
__global__ __launch_bounds__(256) void unpermute_grad_kernel(const UnpermuteParams p, int waves,
                                                             int token_wgs) {
  typedef RowVec<TY, WHOLE> V;
  typedef typename V::raw raw;
  __shared__ float part[4][kAtOnce];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  raw* drows = static_cast<raw*>(p.drows);
  const int64_t vecs = row_vectors(p.cols, V::N);
  if (static_cast<int>(blockIdx.x) >= token_wgs) {
    // 64 rows a wave: those that have no slot
    const int64_t r0 = ((blockIdx.x - token_wgs) * int64_t{4} + wave) * 64;
    uint64_t todo = __ballot(r0 + lane < p.n_rows && p.slot_of_row[r0 + lane] < 0);
    V zero;
#pragma unroll
    for (int c = 0; c < V::N; ++c) zero.set(c, 0.f);
    while (todo) {
      const int64_t r = r0 + __ffsll(static_cast<long long>(todo)) - 1;
      todo &= todo - 1;
      for (int64_t i = lane; i < vecs; i += 64)
        zero.store(drows + r * p.cols + vector_at(i, p.cols, V::N));
    }
    return;
  }
  const int64_t t = blockIdx.x * int64_t{4 / waves} + wave / waves;
  const int sub = wave % waves;
  const bool live = t < p.m;  // (the barriers below are the whole workgroup's)
  const raw* rows = static_cast<const raw*>(p.rows);
  const raw* dout = static_cast<const raw*>(p.dout);
  for (int k0 = 0; k0 < p.topk; k0 += kAtOnce) {
    int64_t row[kAtOnce];
    float w[kAtOnce], dot[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int64_t s = t * p.topk + min(k0 + j, p.topk - 1);
      row[j] = live && k0 + j < p.topk ? p.row_of_slot[s] : -1;
      if (row[j] >= p.n_rows) row[j] = -1;
      w[j] = live && p.weights ? p.weights[s] : 1.f;
      dot[j] = 0.f;
    }
    if (live)
      for (int64_t i = sub * 64 + lane; i < vecs; i += 64 * waves) {
        const int64_t at = vector_at(i, p.cols, V::N);
        const int dup = static_cast<int>(i * V::N - at);  // values the vector before has
        V d, v[kAtOnce];
        d.load(dout + t * p.ldd + at);
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j)
          if (p.dweights && row[j] >= 0) v[j].load(rows + row[j] * p.ld + at);
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
          if (row[j] < 0) continue;
          if (p.dweights)
#pragma unroll
            for (int c = 0; c < V::N; ++c)
              dot[j] = c >= dup ? __builtin_fmaf(d[c], v[j][c], dot[j]) : dot[j];
          if (drows) {
            V o;
#pragma unroll
            for (int c = 0; c < V::N; ++c) o.set(c, w[j] * d[c]);
            o.store(drows + row[j] * p.cols + at);
          }
        }
      }
    if (p.dweights) {
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) dot[j] = wave_sum_f32(dot[j]);
      __syncthreads();
      if (lane == 0)
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) part[wave][j] = dot[j];
      __syncthreads();
      const int k = k0 + lane;
      if (live && sub == 0 && lane < kAtOnce && k < p.topk) {
        float s = 0.f;
        for (int q = 0; q < waves; ++q) s += part[wave + q][lane];
        p.dweights[t * p.topk + k] = s;
      }
    }
  }
}

template <int TY, bool WHOLE>
static int unpermute_width(const UnpermuteParams& p, hipStream_t stream) {
  constexpr int N = RowVec<TY, WHOLE>::N;
  const int64_t vecs = row_vectors(p.cols, N);
  if (!p.out) {
    // a wave a token, or all four for rows of more than 256 vectors
    const int waves = vecs > 256 ? 4 : 1;
    const int64_t tokens = (p.m * waves + 3) / 4;
    const int64_t tail = p.drows ? (p.n_rows + 255) / 256 : 0;
    if (tokens + tail > 0xffffffll) return fail(FGS_EUNSUPPORTED, "too many rows for a grid");
    if (tokens + tail == 0) return FGS_OK;
    hipLaunchKernelGGL((unpermute_grad_kernel<TY, WHOLE>),
                       dim3(static_cast<unsigned>(tokens + tail)), dim3(256), 0, stream, p, waves,
                       static_cast<int>(tokens));
    return check_launch("unpermute_grad_kernel");
  }
  const int l = token_lanes_log2(vecs);
  const int64_t per = 256 >> l;
  const int64_t tokens = (p.m + per - 1) / per;
  const int64_t chunks = (vecs + (int64_t{1} << l) - 1) >> l;
  if (tokens > 0xffffffll || chunks > 0xffff)
    return fail(FGS_EUNSUPPORTED, "too many rows or columns for a grid");
  auto kernel = p.weights ? unpermute_kernel<TY, WHOLE, true> : unpermute_kernel<TY, WHOLE, false>;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(tokens), static_cast<unsigned>(chunks)),
                     dim3(256), 0, stream, p, l);
  return check_launch("unpermute_kernel");
}
template <int TY>
static int unpermute_type(const UnpermuteParams& p, hipStream_t stream) {
  return p.cols * static_cast<int64_t>(sizeof(typename Elem<TY>::raw)) >= 16
             ? unpermute_width<TY, true>(p, stream)
             : unpermute_width<TY, false>(p, stream);
}
int launch_unpermute(const UnpermuteParams& p, int dtype, hipStream_t stream) {
  switch (dtype) {
    case FGS_DTYPE_BF16: return unpermute_type<FGS_DTYPE_BF16>(p, stream);
    case FGS_DTYPE_FP16: return unpermute_type<FGS_DTYPE_FP16>(p, stream);
    default: return unpermute_type<FGS_DTYPE_FP32>(p, stream);
  }
}

}  // namespace fgs

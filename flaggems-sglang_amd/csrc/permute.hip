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
// Memory words at any address. Rows that are written leave with non-temporal stores:
// they are not read again before the caches have turned over (8192 tokens of 4 KB to
// eight rows each 49 us, 52 without).
typedef uint32_t Unaligned128 __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t Unaligned32 __attribute__((aligned(1)));
template <int W>
struct WordOf;
template <>
struct WordOf<16> {
  typedef Unaligned128 type;
};
template <>
struct WordOf<4> {
  typedef Unaligned32 type;
};
template <>
struct WordOf<2> {
  typedef uint16_t type;
};
template <>
struct WordOf<1> {
  typedef uint8_t type;
};

// Sixteen bytes (or one value, for rows shorter than that).
template <int TY, bool WHOLE>
struct RowVec {
  typedef typename Elem<TY>::raw raw;
  static constexpr int N = WHOLE ? 16 / sizeof(raw) : 1;
  typedef typename WordOf<WHOLE ? 16 : sizeof(raw)>::type Word;
  raw v[N];
  __device__ __forceinline__ void load(const void* p) {
    const Word w = *static_cast<const Word*>(p);
    __builtin_memcpy(v, &w, sizeof(v));
  }
  __device__ __forceinline__ void store(void* p) const {
    Word w;
    __builtin_memcpy(&w, v, sizeof(v));
    __builtin_nontemporal_store(w, static_cast<Word*>(p));
  }
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

// A value that is the same in all lanes, as a scalar.
template <bool SAME>
__device__ __forceinline__ int uniform(int v) {
  return SAME ? __builtin_amdgcn_readfirstlane(v) : v;
}

// Threads a token takes: a power of two, at most a workgroup.
static int token_lanes_log2(int64_t vectors) {
  int l = 0;
  while (l < 8 && (int64_t{1} << l) < vectors) ++l;
  return l;
}

constexpr int kAtOnce = 8;    // slots whose rows a thread has in flight
constexpr int kTailRows = 4;  // rows a wave looks at for those without a slot

// ---------------------------------------------------------- tokens -> rows ---
// rows[row of (t, k)] = x[t] (as bytes). With the ids, the row of a slot that no
// expert here has is one behind all experts' and gets zeros, and the order's final
// form is written; without, such a slot has no row (-1), and the workgroups behind
// the tokens' clear the rows that have no slot.
template <int W, bool WAVES>
__global__ __launch_bounds__(256) void permute_kernel(const PermuteParams p, int lanes_log2,
                                                      int token_wgs) {
  typedef typename WordOf<W>::type Word;
  const int lanes = 1 << lanes_log2;
  auto put = [](uint8_t* to, Word v) {
    __builtin_nontemporal_store(v, reinterpret_cast<Word*>(to));
  };
  if (static_cast<int>(blockIdx.x) >= token_wgs) {
    const int64_t r0 = ((blockIdx.x - token_wgs) * int64_t{4} + uniform<true>(threadIdx.x >> 6)) *
                       kTailRows;
    for (int64_t r = r0; r < min(r0 + kTailRows, p.m * p.topk); ++r) {
      if (p.slot_of_row[r] >= 0) continue;
      for (int64_t i = (threadIdx.x & 63) + blockIdx.y * int64_t{64}; i < row_vectors(p.bytes, W);
           i += gridDim.y * int64_t{64})
        put(p.rows + r * p.bytes + vector_at(i, p.bytes, W), Word{});
    }
    return;
  }
  const int64_t t = blockIdx.x * int64_t{256 >> lanes_log2} +
                    uniform<WAVES>(threadIdx.x >> lanes_log2);
  if (t >= p.m) return;
  const int64_t i = (threadIdx.x & (lanes - 1)) + blockIdx.y * int64_t{lanes};
  if (i >= row_vectors(p.bytes, W)) return;
  const int64_t at = vector_at(i, p.bytes, W);
  const Word v = *reinterpret_cast<const Word*>(p.x + t * p.x_stride + at);
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
      put(p.rows + row[j] * p.bytes + at, kept ? v : Word{});
    }
  }
}

// The same for up to 64 slots, with the order: a decode step's, for which a launch of
// its own takes as long as the rows do (8 slots of 256 experts, 7168 columns 10.7 us in
// two launches, 7.4 so). Every wave finds all slots' places, a slot a lane: ballots
// over the bits of the experts' numbers, most significant first, give the lanes of an
// equal and of a smaller one.
template <int W>
__global__ __launch_bounds__(256) void permute_few_kernel(const PermuteParams p, int lanes_log2,
                                                          int id_bits) {
  typedef typename WordOf<W>::type Word;
  const int lane = threadIdx.x & 63, lanes = 1 << lanes_log2;
  const int slots = static_cast<int>(p.m) * p.topk;
  const bool slot = lane < slots;
  const int id = slot ? p.ids[lane] : -1;
  const bool kept = id >= 0 && id < p.experts;
  const int e = kept ? id : p.experts;
  uint64_t eq = __ballot(slot), lt = 0;
  for (int b = id_bits - 1; b >= 0; --b) {
    const bool bit = slot && ((e >> b) & 1);
    const uint64_t on = __ballot(bit);
    if (bit) lt |= eq & ~on;
    eq &= bit ? on : ~on;
  }
  const uint64_t below = lane ? ~0ull >> (64 - lane) : 0;
  const int place = __popcll(lt) + __popcll(eq & below);
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < 64) {
    for (int q = lane; q < p.experts; q += 64) p.counts[q] = 0;
    // the zeros are written before the counts
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_s_waitcnt(0);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (kept && (eq & below) == 0) p.counts[e] = __popcll(eq);
    if (slot) {
      p.row_of_slot[lane] = kept ? place : -1;
      p.slot_of_row[place] = kept ? lane : -1;
    }
  }
  const int t = blockIdx.x * (256 >> lanes_log2) + (threadIdx.x >> lanes_log2);
  const int64_t i = (threadIdx.x & (lanes - 1)) + blockIdx.y * int64_t{lanes};
  const bool mine = t < p.m && i < row_vectors(p.bytes, W);
  const int64_t at = vector_at(i, p.bytes, W);
  Word v{};
  if (mine) v = *reinterpret_cast<const Word*>(p.x + t * p.x_stride + at);
  for (int k = 0; k < p.topk; ++k) {
    const int from = min(t * p.topk + k, 63);  // (whole waves shuffle)
    const int64_t row = __shfl(place, from, 64);
    const bool has = __shfl(static_cast<int>(kept), from, 64);
    if (mine)
      __builtin_nontemporal_store(has ? v : Word{},
                                  reinterpret_cast<Word*>(p.rows + row * p.bytes + at));
  }
}
template <int W>
static int permute_few(const PermuteParams& p, hipStream_t stream) {
  const int64_t vecs = row_vectors(p.bytes, W);
  const int l = token_lanes_log2(vecs);
  const int per = 256 >> l;
  int id_bits = 0;
  while ((1 << id_bits) <= p.experts) ++id_bits;
  hipLaunchKernelGGL(permute_few_kernel<W>,
                     dim3(static_cast<unsigned>((p.m + per - 1) / per),
                          static_cast<unsigned>((vecs + (int64_t{1} << l) - 1) >> l)),
                     dim3(256), 0, stream, p, l, id_bits);
  return check_launch("permute_few_kernel");
}
int launch_permute_few(const PermuteParams& p, hipStream_t stream) {
  if (p.bytes >= 16) return permute_few<16>(p, stream);
  if (p.bytes >= 4) return permute_few<4>(p, stream);
  return permute_few<1>(p, stream);
}

template <int W>
static int permute_width(const PermuteParams& p, hipStream_t stream) {
  const int64_t vecs = row_vectors(p.bytes, W);
  const int l = token_lanes_log2(vecs);
  const int64_t per = 256 >> l;
  const int64_t tokens = (p.m + per - 1) / per;
  const int64_t tail = p.ids ? 0 : (p.m * p.topk + 4 * kTailRows - 1) / (4 * kTailRows);
  const int64_t chunks = (vecs + (int64_t{1} << l) - 1) >> l;
  if (tokens + tail > 0xffffffll || chunks > 0xffff)
    return fail(FGS_EUNSUPPORTED, "too many rows or columns for a grid");
  auto kernel = l >= 6 ? permute_kernel<W, true> : permute_kernel<W, false>;
  hipLaunchKernelGGL(kernel,
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
// without a row (outside [0, n_rows)) adds nothing, whatever its weight is. Bound by
// the rows' bytes (8192 tokens of eight 4 KB rows 47-54 us, 5.6-6.4 TB/s).
// WAVES: a token has whole waves, so its slots' rows and weights are scalars.
template <int TY, bool WHOLE, bool WEIGHTS, bool WAVES>
__global__ __launch_bounds__(256) void unpermute_kernel(const UnpermuteParams p, int lanes_log2) {
  typedef RowVec<TY, WHOLE> V;
  typedef typename V::raw raw;
  const int lanes = 1 << lanes_log2;
  const int64_t t = blockIdx.x * int64_t{256 >> lanes_log2} +
                    uniform<WAVES>(threadIdx.x >> lanes_log2);
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
// over the waves, always in the same order. Bound by the rows' bytes, read and written
// (4093 tokens of eight 14 KB rows, a quarter of them dropped, 175 us, 5.0 TB/s).
template <int TY, bool WHOLE>
__global__ __launch_bounds__(256) void unpermute_grad_kernel(const UnpermuteParams p, int waves,
                                                             int token_wgs) {
  typedef RowVec<TY, WHOLE> V;
  typedef typename V::raw raw;
  __shared__ float part[4][kAtOnce];
  const int lane = threadIdx.x & 63, wave = uniform<true>(threadIdx.x >> 6);
  raw* drows = static_cast<raw*>(p.drows);
  const int64_t vecs = row_vectors(p.cols, V::N);
  if (static_cast<int>(blockIdx.x) >= token_wgs) {
    // kTailRows rows a wave: those that have no slot
    const int64_t r0 = ((blockIdx.x - token_wgs) * int64_t{4} + wave) * kTailRows;
    V zero;
#pragma unroll
    for (int c = 0; c < V::N; ++c) zero.set(c, 0.f);
    for (int64_t r = r0; r < min(r0 + kTailRows, p.n_rows); ++r) {
      if (p.slot_of_row[r] >= 0) continue;
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
    // a vector a lane, with up to four waves a token
    const int waves = vecs > 128 ? 4 : vecs > 64 ? 2 : 1;
    const int64_t tokens = (p.m * waves + 3) / 4;
    const int64_t tail = p.drows ? (p.n_rows + 4 * kTailRows - 1) / (4 * kTailRows) : 0;
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
  auto kernel = l >= 6 ? (p.weights ? unpermute_kernel<TY, WHOLE, true, true>
                                    : unpermute_kernel<TY, WHOLE, false, true>)
                       : (p.weights ? unpermute_kernel<TY, WHOLE, true, false>
                                    : unpermute_kernel<TY, WHOLE, false, false>);
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

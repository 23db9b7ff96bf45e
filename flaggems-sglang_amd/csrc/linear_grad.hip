// What the products' gradients need beside products: the activation's gradient
// and the bias's.
#include "linear_common.h"

namespace fgs {

// dz = dout act'(z), or for z = [gate | up] dgate = dout up act'(gate), dup = dout
// act(gate): eight columns a thread, bound by its bytes (dout and z read, dz
// written: 8192 x 14336 gated 304 us, 5.4 TB/s). REST: what dz's rounding leaves goes to
// a second matrix, in bf16 whatever dz's type (fp16's range ends near the rests of small
// values), so that the bias's sums are of values good to 16 bits and not of dz's 8
// (366 us; dbias's error against 64 bits is then its last rounding's).
template <int TY, int ACT, bool GATED, bool REST>
__global__ __launch_bounds__(256) void linear_act_grad_kernel(const LinearActGradParams p,
                                                             int64_t vecs, int per_row) {
  const int64_t i = blockIdx.x * int64_t{256} + threadIdx.x;
  if (i >= vecs) return;
  const int64_t r = i / per_row;
  const int64_t c = (i - r * per_row) * 8;
  const int64_t wide = GATED ? 2 * p.n : p.n;
  Vec8<TY, true> d;
  Vec8<FGS_DTYPE_FP32, true> g, u;
  d.load(p.dout, r * p.ldd + c, 8);
  g.load(p.z, r * wide + c, 8);
  if constexpr (GATED) u.load(p.z, r * wide + p.n + c, 8);
  float dg[8], du[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float slope;
    const float a = linear_act_slope<ACT>(g[j], &slope);
    if constexpr (GATED) {
      dg[j] = d[j] * u[j] * slope;
      du[j] = d[j] * a;
    } else {
      dg[j] = d[j] * slope;
    }
  }
  auto put = [&](int64_t at, const float (&v)[8]) {
    store8<TY, true>(p.dz, at, 8, v);
    if constexpr (REST) {
      float rest[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float rounded = Elem<TY>::to_f32(Elem<TY>::from_f32(v[j]));
        rest[j] = fabsf(rounded) < INFINITY ? v[j] - rounded : 0.f;  // (none of what is past the type)
      }
      store8<FGS_DTYPE_BF16, true>(p.rest, at, 8, rest);
    }
  };
  put(r * wide + c, dg);
  if constexpr (GATED) put(r * wide + p.n + c, du);
}

template <int TY>
static int act_grad_type(const LinearActGradParams& p, hipStream_t stream) {
  const int per_row = static_cast<int>(p.n / 8);
  const int64_t vecs = p.rows * per_row;
  const int64_t wgs = (vecs + 255) / 256;
  if (wgs > 0xffffffll) return fail(FGS_EUNSUPPORTED, "too many values for a grid");
  return with_act(p.act, [&](auto act_c) {
    constexpr int ACT = decltype(act_c)::value;
    auto kernel = p.gated ? (p.rest ? linear_act_grad_kernel<TY, ACT, true, true>
                                    : linear_act_grad_kernel<TY, ACT, true, false>)
                          : (p.rest ? linear_act_grad_kernel<TY, ACT, false, true>
                                    : linear_act_grad_kernel<TY, ACT, false, false>);
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(wgs)), dim3(256), 0, stream, p, vecs,
                       per_row);
    return check_launch("linear_act_grad_kernel");
  });
}
int launch_linear_act_grad(const LinearActGradParams& p, int dtype, hipStream_t stream) {
  if (p.rows == 0) return FGS_OK;
  return dtype == FGS_DTYPE_BF16 ? act_grad_type<FGS_DTYPE_BF16>(p, stream)
                                 : act_grad_type<FGS_DTYPE_FP16>(p, stream);
}

// Column sums of a group's rows in fp32: a workgroup has 64 columns (a cache line of
// each row) of a part of the rows, 32 rows at a time and four of those in flight,
// added up in a fixed order. Bound by dz's bytes: 8192 x 28672 99 us, 4.7 TB/s (160
// with 32 columns, whose lines two XCDs read); 65536 x 2048 56 (84 with one row in
// flight), 128 groups of them 53.
// REST: with what dz's rounding left (191 us, 4.9 TB/s; 128 groups 76).
template <int TY, bool REST>
__global__ __launch_bounds__(256) void linear_bias_grad_kernel(const LinearBiasGradParams p) {
  constexpr int AT_ONCE = 4;  // rows that a thread has in flight
  __shared__ float sums[32][65];
  const int e = blockIdx.y, part = blockIdx.z;
  int first = 0, n = p.rows;
  if (p.counts) GroupScan{p.counts, p.groups, p.rows}.range(e, &first, &n);
  const int per = (n + p.parts - 1) / p.parts;
  const int r0 = min(part * per, n), r1 = min(r0 + per, n);
  const int lr = threadIdx.x >> 3, lc = (threadIdx.x & 7) * 8;
  const int64_t col = blockIdx.x * int64_t{64} + lc;
  float acc[8] = {};
  if (col < p.n)
    for (int r = r0 + lr; r < r1; r += 32 * AT_ONCE) {
      Vec8<TY, true> v[AT_ONCE];
      Vec8<FGS_DTYPE_BF16, true> rest[REST ? AT_ONCE : 1];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u)
        if (r + 32 * u < r1) {
          const int64_t at = (static_cast<int64_t>(first) + r + 32 * u) * p.ldd + col;
          v[u].load(p.dz, at, 8);
          if constexpr (REST) rest[u].load(p.rest, at, 8);
        }
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u)
        if (r + 32 * u < r1)
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[j] += REST ? v[u][j] + rest[REST ? u : 0][j] : v[u][j];
    }
#pragma unroll
  for (int j = 0; j < 8; ++j) sums[lr][lc + j] = acc[j];
  __syncthreads();
  for (int half = 16; half > 0; half >>= 1) {
    for (int i = threadIdx.x; i < half * 64; i += 256)
      sums[i >> 6][i & 63] += sums[(i >> 6) + half][i & 63];
    __syncthreads();
  }
  const int64_t c = blockIdx.x * int64_t{64} + threadIdx.x;
  if (threadIdx.x < 64 && c < p.n) {
    const float v = sums[0][threadIdx.x];
    const int64_t at = static_cast<int64_t>(e) * p.n + c;
    if (p.parts > 1) p.part[static_cast<int64_t>(part) * p.groups * p.n + at] = v;
    else static_cast<typename Elem<TY>::raw*>(p.out)[at] = Elem<TY>::from_f32(v);
  }
}
template <int TY>
__global__ __launch_bounds__(256) void linear_bias_join_kernel(const LinearBiasGradParams p,
                                                              int64_t values) {
  const int64_t i = blockIdx.x * int64_t{256} + threadIdx.x;
  if (i >= values) return;
  float v = 0.f;
  for (int k = 0; k < p.parts; ++k) v += p.part[k * values + i];
  static_cast<typename Elem<TY>::raw*>(p.out)[i] = Elem<TY>::from_f32(v);
}

// Parts that give every CU a workgroup or two, none below 256 rows of an even
// group.
int linear_bias_parts(int64_t groups, int64_t rows, int64_t n) {
  const int64_t wgs = groups * ((n + 63) / 64);
  const int64_t want = (512 + wgs - 1) / wgs, most = rows / groups / 256;
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, most, 64})));
}

template <int TY>
static int bias_grad_type(const LinearBiasGradParams& p, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>((p.n + 63) / 64), static_cast<unsigned>(p.groups),
                  static_cast<unsigned>(p.parts));
  auto kernel = p.rest ? linear_bias_grad_kernel<TY, true> : linear_bias_grad_kernel<TY, false>;
  hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, p);
  int rc = check_launch("linear_bias_grad_kernel");
  if (rc || p.parts == 1) return rc;
  const int64_t values = p.groups * p.n;
  hipLaunchKernelGGL(linear_bias_join_kernel<TY>, dim3(static_cast<unsigned>((values + 255) / 256)),
                     dim3(256), 0, stream, p, values);
  return check_launch("linear_bias_join_kernel");
}
int launch_linear_bias_grad(const LinearBiasGradParams& p, int dtype, hipStream_t stream) {
  return dtype == FGS_DTYPE_BF16 ? bias_grad_type<FGS_DTYPE_BF16>(p, stream)
                                 : bias_grad_type<FGS_DTYPE_FP16>(p, stream);
}

}  // namespace fgs

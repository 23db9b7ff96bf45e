// What the products' gradients need beside products: the activation's gradient
// and the bias's.
#include "linear_common.h"

namespace fgs {

// dz = dout act'(z), or for z = [gate | up] dgate = dout up act'(gate), dup = dout
// act(gate): eight columns a thread, bound by its bytes (dout and z read, dz
// written).
template <int TY, int ACT, bool GATED>
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
  store8<TY, true>(p.dz, r * wide + c, 8, dg);
  if constexpr (GATED) store8<TY, true>(p.dz, r * wide + p.n + c, 8, du);
}

template <int TY>
static int act_grad_type(const LinearActGradParams& p, hipStream_t stream) {
  const int per_row = static_cast<int>(p.n / 8);
  const int64_t vecs = p.rows * per_row;
  const int64_t wgs = (vecs + 255) / 256;
  if (wgs > 0xffffffll) return fail(FGS_EUNSUPPORTED, "too many values for a grid");
  return with_act(p.act, [&](auto act_c) {
    constexpr int ACT = decltype(act_c)::value;
    auto kernel = p.gated ? linear_act_grad_kernel<TY, ACT, true>
                          : linear_act_grad_kernel<TY, ACT, false>;
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

// Column sums of a group's rows in fp32: a workgroup has 32 columns of a part of
// the rows, 64 rows at a time, added up in a fixed order. Bound by dz's bytes.
template <int TY>
__global__ __launch_bounds__(256) void linear_bias_grad_kernel(const LinearBiasGradParams p) {
  __shared__ float sums[64][33];
  const int e = blockIdx.y, part = blockIdx.z;
  int first = 0, n = p.rows;
  if (p.counts) GroupScan{p.counts, p.groups, p.rows}.range(e, &first, &n);
  const int per = (n + p.parts - 1) / p.parts;
  const int r0 = min(part * per, n), r1 = min(r0 + per, n);
  const int lr = threadIdx.x >> 2, lc = (threadIdx.x & 3) * 8;
  const int64_t col = blockIdx.x * int64_t{32} + lc;
  float acc[8] = {};
  if (col < p.n)
    for (int r = r0 + lr; r < r1; r += 64) {
      Vec8<TY, true> v;
      v.load(p.dz, (static_cast<int64_t>(first) + r) * p.ldd + col, 8);
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] += v[j];
    }
#pragma unroll
  for (int j = 0; j < 8; ++j) sums[lr][lc + j] = acc[j];
  __syncthreads();
  for (int half = 32; half > 0; half >>= 1) {
    for (int i = threadIdx.x; i < half * 32; i += 256)
      sums[i >> 5][i & 31] += sums[(i >> 5) + half][i & 31];
    __syncthreads();
  }
  const int64_t c = blockIdx.x * int64_t{32} + threadIdx.x;
  if (threadIdx.x < 32 && c < p.n) {
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
  const int64_t wgs = groups * ((n + 31) / 32);
  const int64_t want = (512 + wgs - 1) / wgs, most = rows / groups / 256;
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, most, 64})));
}

template <int TY>
static int bias_grad_type(const LinearBiasGradParams& p, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>((p.n + 31) / 32), static_cast<unsigned>(p.groups),
                  static_cast<unsigned>(p.parts));
  hipLaunchKernelGGL(linear_bias_grad_kernel<TY>, grid, dim3(256), 0, stream, p);
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

// Dense e4m3 product with a scale for each block of 128:
//   out[m, n] = sum_kb as[m, kb] ws[n / 128, kb] sum_{k in kb} a[m, k] w[n, k]  (+ bias[n])
// a [m, k] with a scale per row and 128 columns, w [n, k] with one per 128x128
// block, sums in fp32.
//
// One v_mfma_f32_16x16x128 covers a whole k block, so its result (from a zero
// accumulator) is the block's sum for 16 weight rows x 16 tokens; the weights
// are the MFMA's row operand, so a lane's four results are four weight rows
// (output columns) of one token and one fp32 factor, as * ws, scales them all:
// four FMAs an MFMA, which the VALU does while the next MFMA runs.
//
// The instruction adds products in groups of eight neighbouring k: within a
// group they are aligned to the largest (sum of the two exponents) and cut
// toward zero 13 bits below it; groups are added in fp32 (measured with single
// products beside a larger one). At worst that is seven cuts of 2^-13 (8.5e-4)
// of each group's largest product: more than half a step of fp16, and without a
// bound in terms of a result whose large products cancel. On normal data it is
// 1.5e-5 of the result at any k, against 3e-2 from the operands' own rounding,
// and hidden by the step of a 16-bit output; an fp32 one would show it and is
// not offered.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <string>

#include "dense_common.h"
#include "gemm_tiled_common.h"

namespace fgs {

// ---------------------------------------------------------------- output ---
// The bias of output column n in two steps, so that what lies between covers
// the load: its bits (columns past the end: the last one's; without a bias 0),
// then their value. The kernels load the bits before their first load into LDS
// and count on that order where they wait for those. (Loaded at the end, the
// bias cost 0.4 to 1.6 us: 333 x 2112 x 1552, 64 x 64 tiles, 9.6 and 11.2.)
__device__ __forceinline__ uint32_t bias_bits(const BlockGemmParams& p, int64_t n) {
  uint32_t bits = 0;
  if (p.bias) {
    n = min(n, p.n - 1);
    bits = p.bias_dtype == FGS_DTYPE_FP32 ? static_cast<const uint32_t*>(p.bias)[n]
                                          : static_cast<const uint16_t*>(p.bias)[n];
  }
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  return bits;
}
__device__ __forceinline__ float bias_value(const BlockGemmParams& p, uint32_t bits) {
  if (p.bias_dtype == FGS_DTYPE_FP32) return __uint_as_float(bits);
  return p.bias_dtype == FGS_DTYPE_BF16 ? Elem<FGS_DTYPE_BF16>::to_f32(bits)
                                        : Elem<FGS_DTYPE_FP16>::to_f32(bits);
}
template <int TY>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (TY == FGS_DTYPE_BF16) return cvt_pk_bf16(lo, hi);
  else return Elem<TY>::from_f32(lo) | static_cast<uint32_t>(Elem<TY>::from_f32(hi)) << 16;
}
// Four neighbouring output columns of a token from element `at` on (`left`:
// columns of them that exist; vec: the address allows one 8-byte store).
template <int TY>
__device__ __forceinline__ void store4(void* out, int64_t at, f32x4 v, int64_t left, bool vec) {
  typedef typename Elem<TY>::raw raw;
  raw* o = static_cast<raw*>(out) + at;
  if (vec && left >= 4) {
    *reinterpret_cast<uint2*>(o) = uint2{pack2<TY>(v[0], v[1]), pack2<TY>(v[2], v[3])};
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < left) o[i] = Elem<TY>::from_f32(v[i]);
}
// out[m, n .. n + 3] = v in the output's type.
__device__ __forceinline__ void write_out(const BlockGemmParams& p, int64_t m, int64_t n, f32x4 v,
                                          bool vec) {
  const int64_t left = p.n - n;
  const int64_t at = m * p.ldo + n;
  if (p.out_dtype == FGS_DTYPE_BF16) store4<FGS_DTYPE_BF16>(p.out, at, v, left, vec);
  else store4<FGS_DTYPE_FP16>(p.out, at, v, left, vec);
}

// One wave-wide buffer load into LDS of 4 bytes a lane. (A global load into LDS
// counts as one that may have gone through LDS: behind one, the compiler waits
// for every LDS read at once instead of counting them.)
__device__ __forceinline__ void lds_dma4_buf(__amdgpu_buffer_rsrc_t rsrc, uint32_t voff,
                                             void* lds_dst) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(
      rsrc, (__attribute__((address_space(3))) void*)(lds_dst), 4, voff, 0, 0, 0);
}

// Position of logical 16-byte chunk c of stage row r: the LDS serves 16 lanes
// (256 bytes, two rows) of a 16-byte read at a time, and the XOR spreads the
// 16 rows that lanes 0-15 read at one chunk over all 16 positions.
__device__ __forceinline__ int swizzled(int r, int c) { return c ^ ((r >> 1) & 7); }

// Workgroup i of a grid runs on XCD i % 8. Its place in an order that gives each
// XCD a contiguous eighth of `total`, so that neighbours share an L2. (The grid
// has no workgroup too many: a check for one, which stands before the other
// arguments are loaded, cost 0.3 us a call.)
__device__ __forceinline__ int xcd_order(int i, int total) {
  const int xcd = i & 7;
  return xcd * (total >> 3) + min(xcd, total & 7) + (i >> 3);
}

// ------------------------------------------------------------- few tokens ---
// A workgroup owns 16 MT tokens x 16 NT weight rows; its KW waves split the k
// blocks into contiguous runs and meet in LDS at the end, added in wave order.
// Each wave streams its own blocks -- both operands' rows and the tokens'
// scales -- through a ring of SLOTS LDS slots that is its alone, so nothing but
// its own load counter orders it: the form is bound by the weights' bytes, and
// the ring keeps enough of them in flight. (Straight from memory into the
// MFMA's registers, a load's neighbouring lanes lie in 16 different rows, and
// the address unit takes them one a cycle: 16 tokens 11.7 us at 4096 x 7168.)
// One token: 4096 x 7168 7.3 us (4.0 TB/s), 14336 x 7168 21.3 (4.8 TB/s).
template <int MT_, int NT_, int KW_, int SLOTS_>
struct SkinnyCfg {
  static constexpr int MT = MT_, NT = NT_, KW = KW_, SLOTS = SLOTS_;
  static constexpr int W_AT = MT * 2048, SC_AT = (MT + NT) * 2048;
  static constexpr int SLOT = SC_AT + 256;  // 64 token scales
  static constexpr int NL = 2 * (MT + NT) + 1;
  static constexpr int LDS = KW * SLOTS * SLOT;
  static_assert(MT <= 4 && 128 % (16 * NT) == 0, "one scale a lane, one weight block");
  static_assert(SLOTS >= 2 && SLOTS <= 3 && (SLOTS - 1) * NL < 64 && LDS + 64 * NT <= 160 * 1024,
                "ring");
  static_assert(KW * MT * NT * 1024 <= LDS, "partial sums");
};

// (Two waves a SIMD also where there is one: with the registers of one the
// compiler puts products into AGPRs, and a move an FMA takes them out again: 333 x
// 2112 x 1552 8.4 us, 8.1 so.)
template <class C>
__global__ __launch_bounds__(C::KW * 64, 2) void block_gemm_skinny_kernel(
    const BlockGemmParams p, int nm, int total) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  __shared__ __attribute__((aligned(16))) float bias[16 * C::NT];
  constexpr int MT = C::MT, NT = C::NT, SLOTS = C::SLOTS;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // column by column, so that the tiles that read the same weight rows share an
  // L2: 333 x 2112 x 1552 (64 x 64 tiles) 8.4 us, 9.5 row by row; one row of
  // tiles, 1 x 4096 x 7168, 7.35, 7.25 without the division
  const int at = xcd_order(blockIdx.x, total);
  const int tn = __builtin_amdgcn_readfirstlane(at / nm), tm = at - tn * nm;
  const int64_t n0 = static_cast<int64_t>(tn) * 16 * NT;
  const int64_t m0 = static_cast<int64_t>(tm) * 16 * MT;
  static_assert(16 * NT <= 64, "the first wave has the bias");
  const uint32_t my_bias = wave == 0 ? bias_bits(p, n0 + lane) : 0;
  const int per = (p.kblocks + C::KW - 1) / C::KW;
  const int kb0 = min(wave * per, p.kblocks);
  const int count = min(per, p.kblocks - kb0);
  const int rows_a = static_cast<int>(min<int64_t>(16 * MT, p.m - m0));
  const int rows_w = static_cast<int>(min<int64_t>(16 * NT, p.n - n0));
  const uint32_t lda = static_cast<uint32_t>(p.lda), ldw = static_cast<uint32_t>(p.ldw);

  // Lane l of a load: row l / 8 of its eight, 16-byte chunk l % 8, at the
  // chunk's swizzled place. A resource ends with the last row's last column:
  // rows past it are not accessed (what their slots hold reaches only results
  // that are not stored), nor is anything behind k in the last row.
  uint8_t* ring = lds + wave * SLOTS * C::SLOT;
  const int lrow = lane >> 3;
  const uint32_t c0 = swizzled(lrow, lane & 7) * 16;  // rows 0-7 of 16; 8-15: chunk ^ 4
  const uint32_t a0 = lrow * lda, w0 = lrow * ldw;
  const uint32_t as0 = lane * static_cast<uint32_t>(p.as_row) * 4;
  auto issue = [&](int i) {
    uint8_t* slot = ring + (i % SLOTS) * C::SLOT;
    const int kb = kb0 + i;
    const uint32_t left = static_cast<uint32_t>(p.k) - kb * 128;
    const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(p.a) + m0 * p.lda + static_cast<int64_t>(kb) * 128, 0,
        static_cast<int>((rows_a - 1) * lda + left), kBufWord3);
    const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(p.w) + n0 * p.ldw + static_cast<int64_t>(kb) * 128, 0,
        static_cast<int>((rows_w - 1) * ldw + left), kBufWord3);
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<float*>(p.a_scale) + m0 * p.as_row + kb * p.as_col, 0,
        static_cast<int>((rows_a - 1) * static_cast<uint32_t>(p.as_row) * 4 + 4), kBufWord3);
#pragma unroll
    for (int j = 0; j < 2 * NT; ++j)
      lds_dma16_buf(rw, w0 + j * 8 * ldw + (c0 ^ (64 * (j & 1))), 0, slot + C::W_AT + j * 1024);
#pragma unroll
    for (int j = 0; j < 2 * MT; ++j)
      lds_dma16_buf(ra, a0 + j * 8 * lda + (c0 ^ (64 * (j & 1))), 0, slot + j * 1024);
    // (rows that lie apart are a cache line a token, which the address unit takes
    // one a cycle: 128 tokens at 4096 x 7168 18.4 us, 15.5 with adjacent ones)
    lds_dma4_buf(rs, as0, slot + C::SC_AT);
  };
  auto wait_stages = [&](int n) {  // at most n later blocks in flight
    if (n >= 2) wait_vmcnt<(SLOTS > 2 ? 2 * C::NL : 0)>();
    else if (n == 1) wait_vmcnt<C::NL>();
    else wait_vmcnt<0>();
  };

  const int r = lane & 15, g = lane >> 4;
  const int off_lo = r * 128 + swizzled(r, g) * 16;
  const int off_hi = r * 128 + swizzled(r, g + 4) * 16;
  auto frag = [&](const uint8_t* at) -> i32x8 {
    const i32x4 lo = *reinterpret_cast<const i32x4*>(at + off_lo);
    const i32x4 hi = *reinterpret_cast<const i32x4*>(at + off_hi);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  // ... of the row's last block, of which only `chunks` lie inside k
  auto cut = [&](i32x8& f, int chunks) {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      f[v] = g < chunks ? f[v] : 0;
      f[4 + v] = g + 4 < chunks ? f[4 + v] : 0;
    }
  };

  f32x4 acc[NT][MT];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[j][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < SLOTS; ++i)
    if (i < count) issue(i);
  // The weight block's scale by a scalar load, a block ahead (a load into LDS for
  // it cost 1 to 3 %: 48 x 7168 x 2048 6.7 us, 6.5 so).
  typedef const __attribute__((address_space(4))) float* scalars;
  const scalars w_scales =
      (scalars)(reinterpret_cast<uintptr_t>(p.w_scale + (n0 >> 7) * p.kblocks + kb0));
  float ws_next = count > 0 ? w_scales[0] : 0.f;
  for (int i = 0; i < count; ++i) {
    wait_stages(min(SLOTS - 1, count - 1 - i));
    const uint8_t* slot = ring + (i % SLOTS) * C::SLOT;
    i32x8 w[NT], x[MT];
    float s[MT];
    const float ws = ws_next;
    ws_next = w_scales[min(i + 1, count - 1)];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      s[t] = *reinterpret_cast<const float*>(slot + C::SC_AT + (t * 16 + r) * 4);
      x[t] = frag(slot + t * 2048);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) w[j] = frag(slot + C::W_AT + j * 2048);
    wait_lgkm0();  // the slot is read: refill it
    if (i + SLOTS < count) issue(i + SLOTS);
    const int chunks = static_cast<int>(p.k / 16) - (kb0 + i) * 8;
    if (chunks < 8) {
#pragma unroll
      for (int t = 0; t < MT; ++t) cut(x[t], chunks);
#pragma unroll
      for (int j = 0; j < NT; ++j) cut(w[j], chunks);
    }
    // the MFMAs of two token tiles ahead of their FMAs
    f32x4 part[NT][MT];
#pragma unroll
    for (int t0 = 0; t0 < MT; t0 += 2) {
#pragma unroll
      for (int t = t0; t < t0 + 2 && t < MT; ++t)
#pragma unroll
        for (int j = 0; j < NT; ++j)
          part[j][t] = mfma16_fp8(w[j], x[t], f32x4{0.f, 0.f, 0.f, 0.f});
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = t0; t < t0 + 2 && t < MT; ++t)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int v = 0; v < 4; ++v)
            acc[j][t][v] = __builtin_fmaf(part[j][t][v], s[t] * ws, acc[j][t][v]);
    }
  }

  __syncthreads();  // the rings are done with
  if (threadIdx.x < 16 * NT) bias[threadIdx.x] = bias_value(p, my_bias);
  f32x4* red = reinterpret_cast<f32x4*>(lds);
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int t = 0; t < MT; ++t) red[(wave * NT * MT + j * MT + t) * 64 + lane] = acc[j][t];
  __syncthreads();
  const bool vec = p.ldo % 4 == 0 && reinterpret_cast<uintptr_t>(p.out) % 8 == 0;
  for (int i = threadIdx.x; i < NT * MT * 64; i += C::KW * 64) {
    f32x4 v = red[i];
#pragma unroll
    for (int k = 1; k < C::KW; ++k) v += red[k * NT * MT * 64 + i];
    const int tile = i >> 6, l = i & 63;
    const int64_t m = m0 + (tile % MT) * 16 + (l & 15);
    const int64_t n = n0 + (tile / MT) * 16 + 4 * (l >> 4);
    v += *reinterpret_cast<const f32x4*>(bias + (tile / MT) * 16 + 4 * (l >> 4));
    if (m < p.m && n < p.n) write_out(p, m, n, v, vec);
  }
}

// ------------------------------------------------------------ many tokens ---
// A workgroup of WM x WN waves owns BM tokens x BN weight rows; both operands'
// rows of a k block (128 bytes each) and the block's scales stream into a ring
// of STAGES LDS slots by LDS-DMA. A wave keeps its tokens' fragments of a
// block in registers and takes its weight rows 16 at a time; an MFMA's four
// FMAs follow three MFMAs behind it. 256 x 256: 4096 x 4096 x 7168 103 us (2.3
// PFLOP/s, MFMA 53 % busy, one round of tiles with its fill and epilogue), 8192 x
// 14336 x 7168 658 (2.6 PFLOP/s, 66 %: the clock falls to 1.7 - 1.9 GHz under
// random data; zeros run 3.5 PFLOP/s).
template <int BM_, int BN_, int WM_, int WN_, int STAGES_, int WPE_>
struct BlockCfg {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, STAGES = STAGES_;
  static constexpr int WPE = WPE_;            // waves a SIMD holds
  static constexpr int NW = WM * WN;
  static constexpr int A_BYTES = BM * 128, W_BYTES = BN * 128;
  static constexpr int SC_OFF = A_BYTES + W_BYTES;
  static constexpr int STAGE = SC_OFF + NW * 256;  // a float slot per lane
  static constexpr int LDS = STAGES * STAGE;
  static constexpr int NLA = BM / 8 / NW, NLW = BN / 8 / NW;  // loads per wave
  static constexpr int NL = NLA + NLW + 1;
  static constexpr int RT = BM / WM / 16, CT = BN / WN / 16;  // 16-wide tiles of a wave
  static_assert(NLA * 8 * NW == BM && NLW * 8 * NW == BN, "whole loads");
  static_assert(128 % (CT * 16) == 0, "a wave's weight rows lie in one scale block");
  static_assert(BN % 128 == 0 || 128 % BN == 0, "scale blocks of a tile");
  static_assert(BM + (BN + 127) / 128 <= NW * 64, "scale slots");
  static_assert(STAGES >= 2 && (STAGES - 1) * NL < 64 && LDS + 4 * BN <= 160 * 1024,
                "ring");
  static_assert(CT % 2 == 0, "fragment pipeline");
};

// Tiles go in bands of kBand token tiles walked column by column, so an XCD's 32
// CUs share a few rows' and columns' operands in its L2.
constexpr int kBand = 4;
__device__ __forceinline__ void block_tile(int at, int nm, int nn, int* tm, int* tn) {
  const int b = at / (kBand * nn);
  const int rem = at - b * kBand * nn;
  const int rows = min(kBand, nm - b * kBand);
  // (the divisions run on the VALU: back to scalars, so that the loops and the
  // buffer resources that follow from them are scalar too)
  *tn = __builtin_amdgcn_readfirstlane(rem / rows);
  *tm = __builtin_amdgcn_readfirstlane(b * kBand + rem % rows);
}

// OUT: the output's type.
template <class C, int OUT>
__global__ __launch_bounds__(C::NW * 64, C::WPE) void block_gemm_tiled_kernel(
    const BlockGemmParams p, int nm, int nn) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  __shared__ __attribute__((aligned(16))) float tile_biases[C::BN];
  constexpr int RT = C::RT, CT = C::CT, STAGES = C::STAGES;
  int tm, tn;
  block_tile(xcd_order(blockIdx.x, nm * nn), nm, nn, &tm, &tn);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / C::WN, wn = wave % C::WN;
  const int64_t m0 = static_cast<int64_t>(tm) * C::BM;
  const int64_t n0 = static_cast<int64_t>(tn) * C::BN;

  static_assert(C::BN <= C::NW * 64 && C::BN % 64 == 0, "a bias a thread");
  const uint32_t my_bias = wave < C::BN / 64 ? bias_bits(p, n0 + threadIdx.x) : 0;

  // this lane's source of each load: row lane / 8, chunk lane % 8, as byte
  // offsets from the tile's first row (rows past the end read the last one;
  // their results are not stored)
  const int lrow = lane >> 3;
  const int am = static_cast<int>(min<int64_t>(C::BM, p.m - m0)) - 1;  // last rows
  const int wm_last = static_cast<int>(min<int64_t>(C::BN, p.n - n0)) - 1;
  const uint32_t lda = static_cast<uint32_t>(p.lda), ldw = static_cast<uint32_t>(p.ldw);
  uint32_t aoff[C::NLA], woff[C::NLW];
#pragma unroll
  for (int i = 0; i < C::NLA; ++i) {
    const int r = (wave * C::NLA + i) * 8 + lrow;
    aoff[i] = min(r, am) * lda + swizzled(r, lane & 7) * 16;
  }
#pragma unroll
  for (int i = 0; i < C::NLW; ++i) {
    const int r = (wave * C::NLW + i) * 8 + lrow;
    woff[i] = min(r, wm_last) * ldw + swizzled(r, lane & 7) * 16;
  }
  // scale slots: a token's each, then the tile's weight blocks' (a wave's 64
  // are all the one or the other)
  static_assert(C::BM % 64 == 0, "scale slots by waves");
  const bool a_slots = wave < C::BM / 64;
  const float* sc_base = a_slots ? p.a_scale + m0 * p.as_row : p.w_scale + (n0 >> 7) * p.kblocks;
  const int64_t sc_step = a_slots ? p.as_col : 1;
  const int w_block = min<int>(wave * 64 + lane - C::BM,
                               min<int>((C::BN + 127) / 128 - 1, wm_last >> 7));
  const uint32_t sc_off = a_slots ? min(wave * 64 + lane, am) * static_cast<uint32_t>(p.as_row) * 4
                                  : max(w_block, 0) * p.kblocks * 4;

  const int KT = p.kblocks;

  // Loads [from, to) of stage kt. The resources start at its columns and end
  // with the tile's last row: what a lane would read past that (the last
  // block's chunks past k of the last row) is not accessed.
  auto issue = [&](int kt, int from, int to) {
    uint8_t* base = lds + (kt % STAGES) * C::STAGE;
    const int64_t koff = static_cast<int64_t>(kt) * 128;
    const uint32_t left = static_cast<uint32_t>(static_cast<int>(p.k) - kt * 128);
    const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(p.a) + m0 * p.lda + koff, 0, static_cast<int>(am * lda + left),
        kBufWord3);
    const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(p.w) + n0 * p.ldw + koff, 0, static_cast<int>(wm_last * ldw + left),
        kBufWord3);
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<float*>(sc_base) + kt * sc_step, 0, 0x7fffffff, kBufWord3);
#pragma unroll
    for (int i = 0; i < C::NL; ++i) {
      if (i < from || i >= to) continue;
      if (i < C::NLA)
        lds_dma16_buf(ra, aoff[i], 0, base + (wave * C::NLA + i) * 1024);
      else if (i < C::NLA + C::NLW)
        lds_dma16_buf(rw, woff[i - C::NLA], 0,
                      base + C::A_BYTES + (wave * C::NLW + i - C::NLA) * 1024);
      else
        lds_dma4_buf(rs, sc_off, base + C::SC_OFF + wave * 256);
    }
  };
  // Stage kt (this wave's loads of it done): where it is the row's last block
  // and k ends inside it, the chunks past k that this wave loaded become 0.
  const int ragged = p.k & 127 ? KT - 1 : -1;
  auto end_of_k = [&](int kt) {
    if (kt != ragged) return;
    uint8_t* base = lds + (kt % STAGES) * C::STAGE + lane * 16;
    const int live = static_cast<int>(p.k & 127) / 16;
#pragma unroll
    for (int i = 0; i < C::NLA; ++i)
      if (swizzled((wave * C::NLA + i) * 8 + lrow, lane & 7) >= live)
        *reinterpret_cast<u32x4*>(base + (wave * C::NLA + i) * 1024) = u32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < C::NLW; ++i)
      if (swizzled((wave * C::NLW + i) * 8 + lrow, lane & 7) >= live)
        *reinterpret_cast<u32x4*>(base + C::A_BYTES + (wave * C::NLW + i) * 1024) =
            u32x4{0, 0, 0, 0};
    wait_lgkm0();
  };
  const int r16 = lane & 15, g = lane >> 4;
  const int off_lo = r16 * 128 + swizzled(r16, g) * 16;
  const int off_hi = r16 * 128 + swizzled(r16, g + 4) * 16;
  const int a_at = wm * RT * 2048, w_at = C::A_BYTES + wn * CT * 2048;
  auto frag = [&](const uint8_t* at) -> i32x8 {
    const i32x4 lo = *reinterpret_cast<const i32x4*>(at + off_lo);
    const i32x4 hi = *reinterpret_cast<const i32x4*>(at + off_hi);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  // a stage's scales: the wave's tokens' and its weight block's
  auto raw_scales = [&](const uint8_t* st, float (&a)[RT], float& w) {
    const float* sc = reinterpret_cast<const float*>(st + C::SC_OFF);
    w = sc[C::BM + wn * CT * 16 / 128];
#pragma unroll
    for (int t = 0; t < RT; ++t) a[t] = sc[wm * RT * 16 + t * 16 + r16];
  };

  f32x4 acc[CT][RT];
#pragma unroll
  for (int i = 0; i < CT; ++i)
#pragma unroll
    for (int t = 0; t < RT; ++t) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};

#pragma unroll
  for (int s = 0; s < STAGES; ++s)
    if (s < KT) issue(s, 0, C::NL);
  if (KT >= STAGES) wait_vmcnt<(STAGES - 1) * C::NL>();
  else wait_vmcnt<0>();
  if (KT == 1) end_of_k(0);
  wave_barrier_all();

  // Tile j = i * RT + t of a stage (16 weight rows i, 16 tokens t): its MFMA is
  // issued LAG tiles ahead of its four FMAs, across the stage's end too (`sp`:
  // the scales of the stage before).
  constexpr int TILES = CT * RT, LAG = 3;
  static_assert(TILES > LAG && RT >= 2, "pipeline");
  static_assert(C::NL - RT <= (CT - 1) * RT && RT <= C::NL,
                "a refill ends before the next barrier");
  i32x8 x[RT], w[2];
  float s[RT], sp[RT];
  f32x4 part[LAG + 1];
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  // (the first stage folds LAG zeros in)
#pragma unroll
  for (int j = 0; j <= LAG; ++j) part[j] = zero;
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    sp[t] = 0.f;
    x[t] = frag(lds + a_at + t * 2048);
  }
  w[0] = frag(lds + w_at);
  float w_scale0;
  raw_scales(lds, s, w_scale0);
#pragma unroll
  for (int t = 0; t < RT; ++t) s[t] *= w_scale0;
  auto fold = [&](int j, const float (&f)[RT]) {
    const int i = j / RT, t = j % RT;
#pragma unroll
    for (int v = 0; v < 4; ++v)
      acc[i][t][v] = __builtin_fmaf(part[j & LAG][v], f[t], acc[i][t][v]);
  };
  // Nothing of the sums so far is computed behind this point.
  auto settle = [&]() {
#pragma unroll
    for (int i = 0; i < CT; ++i)
#pragma unroll
      for (int t = 0; t < RT; ++t) asm volatile("" : "+v"(acc[i][t]));
#pragma unroll
    for (int j = 0; j <= LAG; ++j) asm volatile("" : "+v"(part[j]));
  };
  static_assert((LAG & (LAG + 1)) == 0 && TILES % (LAG + 1) == 0, "part ring");
  // One stage. The last 16 weight rows' fragment is its last read, so the
  // slot is free once every wave has it; the next stage's first fragments
  // replace each token tile's as its last MFMA has been issued.
  // REST: the stages behind this one, as far as it matters (STAGES: a refill
  // of its slot among them; STAGES - 1 and not FIRST: the rest of the refill
  // that the stage before has begun). The loop's body has no branch: code
  // behind one would draw the MFMAs before it in. A refill's loads go out one a
  // tile: all at once, the eight waves' 72 stood before the address unit (16
  // cycles each) and held every MFMA behind them: 8192^3 450 -> 415 us.
  auto stage = [&](int kt, auto rest_c, auto first_c) {
    constexpr int REST = decltype(rest_c)::value;
    constexpr bool FIRST = decltype(first_c)::value;
    constexpr bool MORE = REST > 0;
    constexpr int L = CT - 1;
    const uint8_t* st = lds + (kt % STAGES) * C::STAGE;
    const uint8_t* nx = lds + ((kt + 1) % STAGES) * C::STAGE;
    float sn[RT], swn = 0.f;
#pragma unroll
    for (int j = 0; j < TILES; ++j) {
      const int i = j / RT, t = j % RT;
      if (t == 0 && i < L) w[(i + 1) & 1] = frag(st + w_at + (i + 1) * 2048);
      if constexpr (MORE) {
        if (i == L && t == 0) {
          wait_lgkm0();
          wait_vmcnt<(REST - 1 < STAGES - 2 ? REST - 1 : STAGES - 2) * C::NL>();
          if constexpr (REST == 1) {
            settle();  // (behind end_of_k's branch they would spill)
            end_of_k(kt + 1);
          }
          wave_barrier_all();
        }
      }
      part[j & LAG] = mfma16_fp8(w[i & 1], x[t], zero);
      if (j >= LAG) fold(j - LAG, s);
      else fold(TILES + j - LAG, sp);
      // refills, a load a tile: RT of them behind the barrier, the others at the
      // next stage's start
      if constexpr (REST == STAGES) {
        if (i == L) issue(kt + STAGES, t, t + 1);
      }
      if constexpr (REST >= STAGES - 1 && !FIRST) {
        if (j + RT < C::NL) issue(kt + STAGES - 1, j + RT, j + RT + 1);
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (MORE) {
        if (i == L) {
          if (t == 0) raw_scales(nx, sn, swn);
          x[t] = frag(nx + a_at + t * 2048);
          if (t == 0) w[0] = frag(nx + w_at);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) sp[t] = s[t];
    if constexpr (MORE) {
#pragma unroll
      for (int t = 0; t < RT; ++t) s[t] = sn[t] * swn;
    }
  };
  // (so that the loop's own reads are all there is to count at its head)
  wait_lgkm0();
  const std::false_type later{};
  int kt = 0;
  if (kt + STAGES < KT) {
    stage(kt, std::integral_constant<int, STAGES>{}, std::true_type{});
    ++kt;
    for (; kt + STAGES < KT; ++kt) stage(kt, std::integral_constant<int, STAGES>{}, later);
    // (the refill of the last stage goes on)
    stage(KT - STAGES, std::integral_constant<int, STAGES - 1>{}, later);
  } else if (KT >= STAGES) {
    stage(0, std::integral_constant<int, STAGES - 1>{}, std::true_type{});
  }
  // the stages behind them, of which fewer than STAGES - 1 are left
  auto tail = [&](auto self, auto rest_c) {
    constexpr int REST = decltype(rest_c)::value;
    if constexpr (REST > 0) {
      if (KT > REST) stage(KT - 1 - REST, rest_c, std::true_type{});
      self(self, std::integral_constant<int, REST - 1>{});
    }
  };
  tail(tail, std::integral_constant<int, STAGES - 2>{});
  stage(KT - 1, std::integral_constant<int, 0>{}, std::true_type{});
#pragma unroll
  for (int j = TILES - LAG; j < TILES; ++j) fold(j, sp);
  // Matrix instructions write every lane, whatever EXEC holds: the last stage's
  // may not be moved into the branches of single lanes that store their
  // results, where they would overwrite registers of the lanes outside.
  settle();

  // A lane holds token r16 of each tile, output columns 4 g .. 4 g + 3. They go
  // through this wave's share of the ring, so that 16 bytes a lane leave as
  // whole row segments (stored from here, four columns a lane are 32 bytes of 16
  // rows each: 257 x 257 x 272 took 22 us). A staged row's 16-byte chunks are
  // XORed with the row: the 16 rows a write covers meet all banks.
  constexpr int CH = CT * 2;                 // chunks of a row
  constexpr int ROWS = 64 / CH;              // rows a store instruction covers
  static_assert(RT * 16 * CH * 16 <= C::LDS / C::NW && 64 % CH == 0, "staging area");
  if (threadIdx.x < C::BN) tile_biases[threadIdx.x] = bias_value(p, my_bias);
  __syncthreads();  // and every wave has read its last fragments
  uint8_t* stg = lds + wave * (RT * 16 * CH * 16);
#pragma unroll
  for (int i = 0; i < CT; ++i) {
    const f32x4 bias =
        *reinterpret_cast<const f32x4*>(tile_biases + (wn * CT + i) * 16 + 4 * g);
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const f32x4 v = acc[i][t] + bias;
      const int c = (2 * i + (g >> 1)) ^ (r16 % CH);
      *reinterpret_cast<uint2*>(stg + (t * 16 + r16) * (CH * 16) + c * 16 + (g & 1) * 8) =
          uint2{pack2<OUT>(v[0], v[1]), pack2<OUT>(v[2], v[3])};
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  const bool vec = p.ldo % 8 == 0 && reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
  const int64_t n = n0 + wn * CT * 16 + (lane % CH) * 8;
  uint16_t* out = static_cast<uint16_t*>(p.out) + n;
#pragma unroll
  for (int k = 0; k < RT * 16 / ROWS; ++k) {
    const int row = k * ROWS + lane / CH;
    const int64_t m = m0 + wm * RT * 16 + row;
    const u32x4 v = *reinterpret_cast<const u32x4*>(stg + row * (CH * 16) +
                                                    ((lane % CH) ^ (row % CH)) * 16);
    if (m >= p.m) continue;
    if (vec && n + 8 <= p.n) {
      *reinterpret_cast<u32x4*>(out + m * p.ldo) = v;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (n + j < p.n)
          out[m * p.ldo + j] = static_cast<uint16_t>(v[j / 2] >> (16 * (j & 1)));
    }
  }
}

// ---------------------------------------------------------------- schedule ---
namespace {

// The forms (FGS_BLOCK_FORM(i)): tile in tokens x weight rows; k blocks an
// iteration takes (the streaming forms' waves take one each); workgroups that
// run at once; microseconds of an iteration with the chip full, and beside the
// iterations of a round: fitted to 500 products drawn over m 1 to 8192, n 16 to
// 16384, k 128 to 16384 (the choice takes 1.3 and 0.8 % more than the best form on
// two sets of 200 others).
// Measured at K 7168 and N 4096, weights not in a cache (tokens: us): 1: 7.3
// (form 0), 16: 9.1 (0), 32: 10.6 (1; 12.2 with 32 x 32), 64: 11.8 (2; 16.4 with
// 64 x 32), 128: 15.6 (3; 18.6 with 32 x 32), 256: 19.5 (4; 29 with 64 x 128),
// 512: 30.4 (5; 36 deep 128 x 128), 1024: 41 (7; 55 with the shallow ring),
// 2048: 66 (8; 70 with 128 x 128), 4096: 104 (9; 125 with 128 x 256).
// Between the tiles: an operand passes the L2 once for each tile that shares it
// (13 TB/s beside the products), so a larger tile is faster until too few are
// left for the CUs; a CU that has one workgroup of four waves alone waits for
// each refill, hence the deep ring with eight.
struct Form {
  int bm, bn, step, at_once;
  double iter, half, round;  // half: an iteration with half of at_once or fewer
};
constexpr Form kForms[] = {
    {16, 16, 8, 512, 1.07, 0.85, 0.5},    {32, 16, 8, 256, 1.05, 0.95, 0.5},
    {32, 32, 8, 256, 1.11, 1.03, 0.78},   {64, 32, 4, 256, 0.9, 0.9, 1.0},
    {64, 64, 4, 256, 1.22, 1.13, 1.62},   {64, 128, 1, 512, 0.73, 0.35, 1.95},
    {128, 128, 1, 512, 1.03, 0.80, 3.0},  {128, 128, 1, 256, 0.58, 0.66, 3.74},
    {128, 256, 1, 256, 0.90, 0.84, 5.01}, {256, 256, 1, 256, 1.54, 1.35, 6.53},
};
constexpr int kNumForms = sizeof(kForms) / sizeof(kForms[0]);

template <int F>
struct FormCfg;
template <> struct FormCfg<0> { typedef SkinnyCfg<1, 1, 8, 2> type; };
template <> struct FormCfg<1> { typedef SkinnyCfg<2, 1, 8, 2> type; };
template <> struct FormCfg<2> { typedef SkinnyCfg<2, 2, 8, 2> type; };
template <> struct FormCfg<3> { typedef SkinnyCfg<4, 2, 4, 3> type; };
template <> struct FormCfg<4> { typedef SkinnyCfg<4, 4, 4, 2> type; };
template <> struct FormCfg<5> { typedef BlockCfg<64, 128, 2, 2, 3, 2> type; };
template <> struct FormCfg<6> { typedef BlockCfg<128, 128, 2, 2, 2, 2> type; };
template <> struct FormCfg<7> { typedef BlockCfg<128, 128, 4, 2, 4, 2> type; };
template <> struct FormCfg<8> { typedef BlockCfg<128, 256, 2, 4, 3, 2> type; };
template <> struct FormCfg<9> { typedef BlockCfg<256, 256, 4, 2, 2, 2> type; };

// Launches `kernel` with more than 64 KiB of LDS, which each GPU has to be told
// of once (`told`: a bit a GPU).
template <class... P, class... A>
int launch_wide_lds(const char* name, void (*kernel)(P...), std::atomic<uint64_t>& told,
                    int64_t wgs, int threads, int lds, hipStream_t stream, A... args) {
  // (the runtime counts a grid in 32-bit threads)
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

template <int F>
int skinny_launch(const BlockGemmParams& p, hipStream_t stream) {
  typedef typename FormCfg<F>::type C;
  static_assert(kForms[F].bm == 16 * C::MT && kForms[F].bn == 16 * C::NT && kForms[F].step == C::KW,
                "form table");
  static std::atomic<uint64_t> told{0};
  const int64_t nm = (p.m + 16 * C::MT - 1) / (16 * C::MT);
  const int64_t nn = (p.n + 16 * C::NT - 1) / (16 * C::NT);
  return launch_wide_lds("block_gemm_skinny_kernel", block_gemm_skinny_kernel<C>, told, nm * nn,
                         C::KW * 64, C::LDS, stream, p, static_cast<int>(nm),
                         static_cast<int>(nm * nn));
}

template <int F, int OUT>
int tiled_launch_out(const BlockGemmParams& p, hipStream_t stream) {
  typedef typename FormCfg<F>::type C;
  static_assert(kForms[F].bm == C::BM && kForms[F].bn == C::BN && kForms[F].step == 1,
                "form table");
  static std::atomic<uint64_t> told{0};
  const int64_t nm = (p.m + C::BM - 1) / C::BM, nn = (p.n + C::BN - 1) / C::BN;
  return launch_wide_lds("block_gemm_tiled_kernel", block_gemm_tiled_kernel<C, OUT>, told, nm * nn,
                         C::NW * 64, C::LDS, stream, p, static_cast<int>(nm),
                         static_cast<int>(nn));
}
template <int F>
int tiled_launch(const BlockGemmParams& p, hipStream_t stream) {
  return p.out_dtype == FGS_DTYPE_BF16 ? tiled_launch_out<F, FGS_DTYPE_BF16>(p, stream)
                                       : tiled_launch_out<F, FGS_DTYPE_FP16>(p, stream);
}

}  // namespace

bool block_gemm_flags_ok(int32_t flags) { return flags >= 0 && flags <= kNumForms; }

// The form with the shortest estimate: rounds of the workgroups that run at
// once, each its iterations. A form of more tokens than there are reads nothing
// more for them, so tokens alone rule none out.
int block_gemm_form(int64_t m, int64_t n, int64_t k, int32_t flags) {
  if (flags) return flags - 1;
  const double blocks = static_cast<double>((k + 127) / 128);
  int best = 0;
  double best_us = 0;
  for (int f = 0; f < kNumForms; ++f) {
    const Form& q = kForms[f];
    const int64_t wgs = ((m + q.bm - 1) / q.bm) * ((n + q.bn - 1) / q.bn);
    const int64_t rounds = (wgs + q.at_once - 1) / q.at_once;
    const double iter = wgs <= q.at_once / 2 ? q.half : q.iter;
    const double iters = std::ceil(blocks / q.step);
    const double us = static_cast<double>(rounds) * (iters * iter + q.round);
    if (f == 0 || us < best_us) {
      best = f;
      best_us = us;
    }
  }
  return best;
}

std::string block_gemm_name(int form) {
  const Form& q = kForms[form];
  return (q.step > 1 ? "stream " : "tiled ") + std::to_string(q.bm) + "x" + std::to_string(q.bn) +
         (form == 7 ? " deep" : "");
}

int launch_block_gemm(const BlockGemmParams& p, int form, hipStream_t stream) {
  switch (form) {
    case 0: return skinny_launch<0>(p, stream);
    case 1: return skinny_launch<1>(p, stream);
    case 2: return skinny_launch<2>(p, stream);
    case 3: return skinny_launch<3>(p, stream);
    case 4: return skinny_launch<4>(p, stream);
    case 5: return tiled_launch<5>(p, stream);
    case 6: return tiled_launch<6>(p, stream);
    case 7: return tiled_launch<7>(p, stream);
    case 8: return tiled_launch<8>(p, stream);
    default: return tiled_launch<9>(p, stream);
  }
}

}  // namespace fgs

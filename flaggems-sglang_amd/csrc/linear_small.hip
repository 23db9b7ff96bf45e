// Products of few rows (linear.hip has the others): bound by the weights' bytes,
// not by the matrix instructions.
//
// A workgroup owns 16 MT rows of x and 16 NT weight rows; its KW waves split the
// sums into contiguous runs and meet in LDS at the end, added in wave order. Each
// wave streams its own blocks of 64 sums -- both operands' rows, 128 bytes of each
// -- through a ring of SLOTS LDS slots that is its alone, so nothing but its own
// load counter orders it. The weights are the MFMA's row operand: a lane's four
// results are four adjacent output columns of one row.
#include <algorithm>
#include <atomic>
#include <string>

#include "linear_common.h"

namespace fgs {

template <int MT_, int NT_, int KW_, int SLOTS_>
struct LinearSmall {
  static constexpr int MT = MT_, NT = NT_, KW = KW_, SLOTS = SLOTS_;
  static constexpr int W_AT = MT * 2048, SLOT = (MT + NT) * 2048;
  static constexpr int NL = 2 * (MT + NT);  // loads of a block
  static constexpr int LDS = KW * SLOTS * SLOT;
  static_assert(SLOTS >= 2 && SLOTS <= 4 && (SLOTS - 1) * NL < 64 && LDS <= 160 * 1024, "ring");
  static_assert(KW * MT * NT * 1024 <= LDS, "partial sums");
};

// INPUT_GRAD: out = x w by w's columns -- a block is 64 of its rows, 128 bytes of each,
// which the LDS reads transpose on the way to the registers.
enum { kSmallForward, kSmallGated, kSmallInputGrad };
template <int TY, int MODE, int ACT, class C>
__global__ __launch_bounds__(C::KW * 64, 2) void linear_small_kernel(const LinearParams p, int nm,
                                                                     int total) {
  typedef Mma16<TY> M;
  typedef typename M::Frag Frag;
  typedef typename Elem<TY>::raw raw;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  constexpr int MT = C::MT, NT = C::NT, SLOTS = C::SLOTS;
  constexpr bool GATED = MODE == kSmallGated, ACROSS = MODE == kSmallInputGrad;
  static_assert(!GATED || NT % 2 == 0, "gate and up rows");
  static_assert(!ACROSS || NT == 4, "128 bytes of a row");
  constexpr int TN = GATED ? 8 * NT : 16 * NT;  // output columns
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Workgroup i runs on XCD i % 8, each of which takes a contiguous eighth of the
  // tiles, column by column, so that tiles that read the same weights share an L2.
  // The grid has tiles for any division of the rows into groups: some have no rows.
  const int i0 = blockIdx.x;
  const int at = (i0 & 7) * (total >> 3) + min(i0 & 7, total & 7) + (i0 >> 3);
  const int tn = __builtin_amdgcn_readfirstlane(at / nm);
  const int tm = at - tn * nm;
  int e = 0, first = tm * 16 * MT, rows = min(16 * MT, p.rows - first);
  if (p.counts) GroupScan{p.counts, p.groups, p.rows}.tile(tm, 16 * MT, &e, &first, &rows);
  e = __builtin_amdgcn_readfirstlane(e);
  first = __builtin_amdgcn_readfirstlane(first);
  rows = __builtin_amdgcn_readfirstlane(rows);
  if (rows <= 0) return;
  const bool none = e >= p.groups;  // rows of no group
  const int n0 = tn * TN;
  const int cols = min(TN, p.n - n0);

  const int blocks = none ? 0 : (p.red + 63) / 64;
  const int per = (blocks + C::KW - 1) / C::KW;
  const int kb0 = min(wave * per, blocks);
  const int count = min(per, blocks - kb0);
  const int ldx = static_cast<int>(p.ldq * 2), ldw = static_cast<int>(p.ldp * 2);
  const uint8_t* x0 = static_cast<const uint8_t*>(p.q) + first * p.ldq * 2;
  const uint8_t* w0 = static_cast<const uint8_t*>(p.p) +
                      (none ? 0 : (e * p.p_group + (ACROSS ? n0 : n0 * p.ldp)) * 2);

  // Lane l of a load: row l / 8 of its eight, 16-byte chunk l % 8 at its swizzled
  // place. A resource ends with the last row's last sum; the chunks past the sums' end
  // in other rows are sent outside it. Loads from outside write zeros.
  uint8_t* ring = lds + wave * SLOTS * C::SLOT;
  const int lrow = lane >> 3;
  const int c0 = ((lane & 7) ^ (lrow >> 1)) * 16;  // rows 0-7 of 16; 8-15: chunk ^ 4
  // (across: 32-byte granule g of row r at place g ^ (bit 1 of r, bit 3): a transposing
  // read takes a granule of four consecutive rows, two of them rows 8 apart at a time)
  const int wc = ((((lane & 7) >> 1) ^ ((lane >> 4) & 1)) * 32) + (lane & 1) * 16;
  auto issue = [&](int i) {
    uint8_t* slot = ring + (i % SLOTS) * C::SLOT;
    const int kb = kb0 + i;
    const int left = (p.red - kb * 64) * 2;
    auto resource = [&](const uint8_t* base, int r, int ld) {
      return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base) + kb * int64_t{128}, 0,
                                               (r - 1) * ld + left, kBufWord3);
    };
    const __amdgpu_buffer_rsrc_t rx = resource(x0, rows, ldx);
    if constexpr (ACROSS) {
      const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<uint8_t*>(w0) + kb * int64_t{64} * ldw, 0,
          (min(64, p.red - kb * 64) - 1) * ldw + (p.n - n0) * 2, kBufWord3);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        lds_dma16_buf(rw, (j * 8 + lrow) * ldw + (wc ^ (64 * (j & 1))), 0,
                      slot + C::W_AT + j * 1024);
    } else {
      const __amdgpu_buffer_rsrc_t rw = resource(w0, cols, ldw);
      const __amdgpu_buffer_rsrc_t ru = resource(GATED ? w0 + p.n * p.ldp * 2 : w0, cols, ldw);
#pragma unroll
      for (int j = 0; j < 2 * NT; ++j) {
        const int c = c0 ^ (64 * (j & 1));
        // (gated: 16 gate rows, the 16 up rows of the same columns, ...)
        const int r = (GATED ? (j >> 2) * 16 + (j & 1) * 8 : j * 8) + lrow;
        const uint32_t o = c < left ? static_cast<uint32_t>(r * ldw + c) : 0x80000000u;
        if (GATED && (j & 2)) lds_dma16_buf(ru, o, 0, slot + C::W_AT + j * 1024);
        else lds_dma16_buf(rw, o, 0, slot + C::W_AT + j * 1024);
      }
    }
#pragma unroll
    for (int j = 0; j < 2 * MT; ++j) {
      const int c = c0 ^ (64 * (j & 1));
      const uint32_t o = c < left ? static_cast<uint32_t>((j * 8 + lrow) * ldx + c) : 0x80000000u;
      lds_dma16_buf(rx, o, 0, slot + j * 1024);
    }
  };
  auto wait_blocks = [&](int n) {  // at most n later blocks in flight
    if (n >= 3) wait_vmcnt<(SLOTS > 3 ? 3 * C::NL : 0)>();
    else if (n == 2) wait_vmcnt<(SLOTS > 2 ? 2 * C::NL : 0)>();
    else if (n == 1) wait_vmcnt<C::NL>();
    else wait_vmcnt<0>();
  };
  const int r = lane & 15, g = lane >> 4;
  int off[2];
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) off[kk] = r * 128 + (((g + 4 * kk) ^ ((r >> 1) & 7)) * 16);

  int across[ACROSS ? NT : 1];
  if constexpr (ACROSS)
#pragma unroll
    for (int j = 0; j < NT; ++j)
      across[j] = (8 * g + (r >> 2)) * 128 + (j ^ ((r >> 3) | (g & 1) << 1)) * 32 + (r & 3) * 8;
  auto weights = [&](const uint8_t* w_slot, int j, int kk) -> Frag {
    if constexpr (ACROSS) {
      const uint8_t* a = w_slot + across[j] + kk * 32 * 128;
      const s16x4 lo = read_transposed((LdsWords)(a));
      const s16x4 hi = read_transposed((LdsWords)(a + 4 * 128));
      return __builtin_bit_cast(Frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      return *reinterpret_cast<const Frag*>(w_slot + j * 2048 + off[kk]);
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
  for (int i = 0; i < count; ++i) {
    wait_blocks(min(SLOTS - 1, count - 1 - i));
    const uint8_t* slot = ring + (i % SLOTS) * C::SLOT;
    Frag w[2][NT], x[2][MT];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
        x[kk][t] = *reinterpret_cast<const Frag*>(slot + t * 2048 + off[kk]);
#pragma unroll
      for (int j = 0; j < NT; ++j)
        w[kk][j] = weights(slot + C::W_AT, j, kk);
    }
    wait_lgkm0();  // the slot is read: refill it
    if (i + SLOTS < count) issue(i + SLOTS);
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[j][t] = M::mma16(w[kk][j], x[kk][t], acc[j][t]);
  }

  __syncthreads();  // the rings are done with
  f32x4* red = reinterpret_cast<f32x4*>(lds);
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int t = 0; t < MT; ++t) red[(wave * NT * MT + j * MT + t) * 64 + lane] = acc[j][t];
  __syncthreads();
  // Four columns of a row a thread. (Loads behind the last load into LDS: the counter's
  // waits are done.)
  constexpr int OT = GATED ? NT / 2 : NT;
  const int wide = GATED ? 2 * p.n : p.n;
  auto sum = [&](int tile) {
    f32x4 v = red[tile * 64 + lane];
#pragma unroll
    for (int k = 1; k < C::KW; ++k) v += red[(k * NT * MT + tile) * 64 + lane];
    return v;
  };
  auto four = [](const raw* a, f32x4& v) {
    uint2 w;
    __builtin_memcpy(&w, a, 8);
    v[0] += Elem<TY>::to_f32(static_cast<raw>(w.x));
    v[1] += Elem<TY>::to_f32(static_cast<raw>(w.x >> 16));
    v[2] += Elem<TY>::to_f32(static_cast<raw>(w.y));
    v[3] += Elem<TY>::to_f32(static_cast<raw>(w.y >> 16));
  };
  auto put = [](void* to, int64_t where, f32x4 v) {
    const uint2 w{pack2<TY>(v[0], v[1]), pack2<TY>(v[2], v[3])};
    __builtin_memcpy(static_cast<raw*>(to) + where, &w, 8);
  };
  for (int tile = wave; tile < OT * MT; tile += C::KW) {
    const int j = tile / MT, t = tile % MT;
    const int m = t * 16 + r, n = n0 + j * 16 + 4 * g;
    f32x4 v = sum(GATED ? 2 * j * MT + t : tile), u{0.f, 0.f, 0.f, 0.f};
    if constexpr (GATED) u = sum((2 * j + 1) * MT + t);
    if (m >= rows || n >= p.n) continue;
    if (!ACROSS && p.bias && !none) {
      const raw* b = static_cast<const raw*>(p.bias) + static_cast<int64_t>(e) * wide + n;
      four(b, v);
      if constexpr (GATED) four(b + p.n, u);
    }
    const int64_t row = first + m;
    if constexpr (ACROSS) {
      put(p.out, row * p.n + n, v);
      continue;
    }
    if (p.z) {
      *reinterpret_cast<f32x4*>(p.z + row * wide + n) = v;
      if constexpr (GATED) *reinterpret_cast<f32x4*>(p.z + row * wide + p.n + n) = u;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      v[q] = linear_act<ACT>(v[q]);
      if constexpr (GATED) v[q] *= u[q];
    }
    if (p.residual) four(static_cast<const raw*>(p.residual) + row * p.ldr + n, v);
    put(p.out, row * p.n + n, v);
  }
}

namespace {

template <int TY, int MODE, int ACT, class C>
int launch_cfg(const LinearParams& p, hipStream_t stream) {
  static std::atomic<uint64_t> told{0};
  constexpr int BM = 16 * C::MT, TN = (MODE == kSmallGated ? 8 : 16) * C::NT;
  const int64_t nm = linear_row_tiles(p, BM), nn = (p.n + TN - 1) / TN;
  if (nm * nn > 0x7fffffffll) return fail(FGS_EUNSUPPORTED, "too many tiles for a grid");
  if (const int rc = MODE == kSmallInputGrad ? check_linear_across(p, kLinearDgrad) : FGS_OK) return rc;
  return launch_lds("linear_small_kernel", linear_small_kernel<TY, MODE, ACT, C>, told, nm * nn,
                    C::KW * 64, C::LDS, stream, p, static_cast<int>(nm),
                    static_cast<int>(nm * nn));
}
// CG: the configuration of the gated product
template <int TY, class C, class CG = C>
int launch_forward(const LinearParams& p, bool gated, hipStream_t stream) {
  return with_act(p.act, [&](auto act_c) {
    constexpr int ACT = decltype(act_c)::value;
    return gated ? launch_cfg<TY, kSmallGated, ACT, CG>(p, stream)
                 : launch_cfg<TY, kSmallForward, ACT, C>(p, stream);
  });
}
template <int TY>
int launch_type(const LinearParams& p, int mode, int form, hipStream_t stream) {
  if (mode == kLinearDgrad) {
    switch (form) {
      case 0: return launch_cfg<TY, kSmallInputGrad, 0, LinearSmall<1, 4, 8, 2>>(p, stream);
      case 1: return launch_cfg<TY, kSmallInputGrad, 0, LinearSmall<2, 4, 4, 3>>(p, stream);
      default: return launch_cfg<TY, kSmallInputGrad, 0, LinearSmall<4, 4, 4, 2>>(p, stream);
    }
  }
  const bool gated = mode == kLinearGated;
  switch (form) {
    case 0: return launch_forward<TY, LinearSmall<1, 1, 8, 2>, LinearSmall<1, 2, 8, 2>>(p, gated, stream);
    case 1: return launch_forward<TY, LinearSmall<1, 2, 8, 2>>(p, gated, stream);
    case 2: return launch_forward<TY, LinearSmall<2, 2, 8, 2>>(p, gated, stream);
    case 3: return launch_forward<TY, LinearSmall<4, 2, 4, 3>>(p, gated, stream);
    default: return launch_forward<TY, LinearSmall<4, 4, 4, 2>>(p, gated, stream);
  }
}

}  // namespace

int launch_linear_small(const LinearParams& p, int mode, int dtype, int form,
                        hipStream_t stream) {
  return dtype == FGS_DTYPE_BF16 ? launch_type<FGS_DTYPE_BF16>(p, mode, form, stream)
                                 : launch_type<FGS_DTYPE_FP16>(p, mode, form, stream);
}

}  // namespace fgs

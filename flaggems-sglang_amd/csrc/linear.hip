// Products of 16-bit matrices with fp32 sums, and their gradients, dense or per
// group of rows (the experts' of tokens sorted by expert):
//   out[m, n] = sum_r Q[m, r] P[n, r]
//   forward    Q = x    [rows, k],      P = w[e] [n, k]
//   dx         Q = dz   [rows, n],      P = w[e] by column, [k, n]
//   dw[e]      Q = dz   by column,      P = x by column, r over the group's rows
// An operand whose sums run along its rows ("along") is staged in LDS as rows of
// 64 sums' values; one whose sums run across rows ("across") as 64 rows of the
// tile's columns, which the LDS reads transpose on the way to the registers
// (ds_read_b64_tr_b16): no transposed copy is ever made.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <string>

#include "linear_common.h"

namespace fgs {

// ------------------------------------------------------------------ tiles ---
// A workgroup of 2 x 2 waves owns a T x T tile; a wave (T / 2)^2 of it in
// 32x32x16 MFMAs, P as the row operand: a lane's results are then runs of four
// adjacent output columns of one output row. Stages of KB sums stream into an LDS
// ring by buffer loads. What lies outside an operand -- rows past the tile's, sums
// past the end, stages behind the last -- is outside its buffer resource or sent
// there: such loads write zeros to LDS (measured), so a sum's tail adds 0 * 0
// whatever memory holds there.
// KB 32: five slots for each operand, loads four stages ahead; KB 64: two for Q and
// three for P, two ahead. The longer way ahead covers an L2 miss, which a stage's
// first reader in an XCD always has; but a row of 32 sums is half a cache line, and
// the second request for it costs more than is won where both operands run along
// their rows. (8192^3, KB 32 / 64, MFMA busy: dw 785 / 823 us, 80 / 67 %; dx 801 / 838;
// forward 852 / 834. The clock falls from 1.8 to 1.56 GHz as the MFMAs get busier.)
template <int T_, int KB_>
struct LinearTile {
  static constexpr int T = T_;
  static constexpr int KB = KB_;              // sums a stage
  static constexpr int KK = KB / 16;          // MFMA steps
  static constexpr int NB = T / 64;           // 32-wide blocks of a wave, each way
  static constexpr int SLOT = T * KB * 2;     // bytes of an operand's stage
  static constexpr int NL = SLOT / 4096;      // loads of a wave per operand and stage
  static constexpr int Q_SLOTS = KB == 32 ? 5 : 2, P_SLOTS = KB == 32 ? 5 : 3;
  static constexpr int P_AT = Q_SLOTS * SLOT;
  static constexpr int LDS = (Q_SLOTS + P_SLOTS) * SLOT;
  static constexpr int STAGING = T * T / 2;   // a wave's part in the epilogue, 16 bits
  // A workgroup has several tiles: only where three stages leave room to stage half a
  // tile beside them.
  static constexpr bool ROUNDS = KB == 32;
  static_assert(KB == 32 || KB == 64, "main loops");
  static_assert(4 * STAGING <= LDS && LDS <= 160 * 1024, "LDS");
  // Place of 16-byte chunk c of row r of KB sums: the LDS serves 16 lanes of a
  // 16-byte read at a time, whose 16 rows share a chunk; the XOR spreads them over
  // the places of the rows that 256 bytes hold.
  static __device__ __forceinline__ int chunk(int r, int c) {
    return c ^ ((r / (128 / KB)) & (KB / 8 - 1));
  }
};

// Offset that no buffer resource here reaches.
constexpr uint32_t kOutside = 0x80000000u;

// Where lane l's 16 bytes of the wave's load i come from, in bytes from the
// stage's origin (`along`: row r of the tile, swizzled chunk of its sums; `across`:
// row of the stage's sums, swizzled chunk of its T columns).
// Across: a transposing read of 16 lanes takes 32 bytes of four consecutive rows;
// the XOR by 2 (row % 4) on 32-byte granules spreads two such reads over 256 bytes.
template <class C, bool ACROSS>
struct Feed {
  uint32_t off[C::NL];
  int c0;  // along: byte in the row of even loads; odd ones: ^ flip
  static constexpr int FLIP = C::KB == 64 ? 64 : 0;

  // row(i): the operand's row, from the tile's first, of the tile's row i
  template <class R>
  __device__ __forceinline__ void init(int wave, int lane, int64_t ld_bytes, R&& row) {
    const uint32_t ld = static_cast<uint32_t>(ld_bytes);
    if constexpr (ACROSS) {
      constexpr int LPR = C::T / 8;      // lanes a row takes
      constexpr int RPL = 64 / LPR;      // rows a load covers
      const int sub = lane / LPR, chunk = lane % LPR;
#pragma unroll
      for (int i = 0; i < C::NL; ++i) {
        const int k = (wave * C::NL + i) * RPL + sub;
        const int granule = (chunk >> 1) ^ (2 * (k & 3));
        off[i] = k * ld + granule * 32 + (chunk & 1) * 16;
      }
      c0 = 0;
    } else {
      constexpr int LPR = C::KB / 8, RPL = 64 / LPR;
      c0 = C::chunk(lane / LPR, lane % LPR) * 16;
#pragma unroll
      for (int i = 0; i < C::NL; ++i)
        off[i] = row((wave * C::NL + i) * RPL + lane / LPR) * ld + (c0 ^ ((i & 1) * FLIP));
    }
  }
};

// The epilogue's staging, which no load in flight writes (__restrict__: as the
// transposing reads).
__device__ __forceinline__ void put_staged(uint2* __restrict__ at, uint2 v) { *at = v; }
__device__ __forceinline__ u32x4 staged(const u32x4* __restrict__ at) { return *at; }

// Tiles of an XCD, and those of its last round that are cut off: of the 32 CUs at most
// half have one, and there is a round before it.
__device__ __host__ __forceinline__ int linear_share(int total, int xcd) {
  return (total >> 3) + (xcd < (total & 7));
}
__device__ __host__ __forceinline__ int linear_rest(int share) {
  const int rest = share & 31;
  return share > 32 && rest <= 16 ? rest : 0;
}

template <int TY, int MODE, int ACT, class C>
__global__ __launch_bounds__(256, 1) void linear_tile_kernel(const LinearParams p) {
  typedef Mma16<TY> M;
  typedef typename M::Frag Frag;
  typedef typename Elem<TY>::raw raw;
  constexpr bool QA = MODE == kLinearWgrad;                          // Q across
  constexpr bool PA = MODE == kLinearWgrad || MODE == kLinearDgrad;  // P across
  constexpr bool GATED = MODE == kLinearGated;
  constexpr bool FORWARD = MODE == kLinearForward || GATED;
  constexpr int T = C::T, NB = C::NB, NL = C::NL, SLOT = C::SLOT;
  constexpr int TN = GATED ? T / 2 : T;  // output columns of a tile
  constexpr int P_AT = C::P_AT, KB = C::KB;
  constexpr bool ROUNDS = C::ROUNDS;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1;

  // ---- the tile. Workgroup b runs on XCD b % 8; each XCD takes a contiguous
  // eighth of the tiles, which go in bands of four columns, row by row, so that
  // the tiles an XCD's 32 CUs have at a time share rows and columns in its L2.
  // A last round that leaves half of the CUs or more without a tile is cut off
  // (kLinearCut) and goes to a second launch in quarters, 128 x 128 (kLinearRest): 36
  // row tiles of 16 columns, 2.25 rounds, k 14336: 975 us in one launch, 932 in two;
  // 4608 x 4096 x 4096 (288 tiles) 215 and 143.
  // ROUNDS: a CU's workgroup takes every 32nd of its XCD's tiles. The next tile's first
  // stages are loaded before a tile is stored, and the stores run on under the first
  // stages' products (128 groups of 65536 rows, 1536 x 2048: dw 545 us with a workgroup
  // a tile, 471 so; dx 496 and 476; 8192^3 level).
  const int quarters = T == 128 && p.part == kLinearRest ? 2 : 1;  // a side
  const int bt = T * quarters, btn = TN * quarters;
  const int n_ct = (p.n + btn - 1) / btn;
  const GroupScan scan{p.counts, p.groups, p.rows};
  const int n_rt = QA ? (p.m + bt - 1) / bt
                      : p.counts ? scan.tiles(bt) : (p.rows + bt - 1) / bt;
  const int total = (QA ? p.groups : 1) * n_rt * n_ct;
  const int xcd = blockIdx.x & 7;
  const int share = linear_share(total, xcd);
  const int rest = p.part == kLinearWhole ? 0 : linear_rest(share);
  int e, rt, ct, first, nrows;  // the tile's: rows of Q [first, first + nrows)
  // Tile (of the XCD's) pos; false if there is none.
  auto locate = [&](int pos) -> bool {
    int sub = 0;
    if (quarters == 2) {
      sub = pos & 3;
      pos = share - rest + (pos >> 2);
      if (pos >= share) return false;
    } else if (pos >= share - rest) {
      return false;
    }
    int at = xcd * (total >> 3) + min(xcd, total & 7) + pos;
    e = 0;
    if (QA) {
      e = at / (n_rt * n_ct);
      at -= e * n_rt * n_ct;
    }
    constexpr int BAND = 4;
    const int band = at / (n_rt * BAND);
    const int cols = min(BAND, n_ct - band * BAND);
    at -= band * n_rt * BAND;
    rt = __builtin_amdgcn_readfirstlane(at / cols);
    ct = __builtin_amdgcn_readfirstlane((band * BAND + at % cols) * quarters + (sub & 1));
    e = __builtin_amdgcn_readfirstlane(e);
    // (across: rows of the group's sums)
    if (!p.counts) {
      first = QA ? 0 : rt * bt;
      nrows = QA ? p.rows : min(bt, p.rows - first);
    } else if (QA) {
      scan.range(e, &first, &nrows);
    } else {
      scan.tile(rt, bt, &e, &first, &nrows);
    }
    rt = rt * quarters + (sub >> 1);
    if (!QA && quarters == 2) {
      first += (sub >> 1) * T;
      nrows = min(T, nrows - (sub >> 1) * T);
    }
    e = __builtin_amdgcn_readfirstlane(e);
    first = __builtin_amdgcn_readfirstlane(first);
    nrows = __builtin_amdgcn_readfirstlane(nrows);
    return ct * TN < p.n && (QA ? rt * T < p.m : nrows > 0);  // (quarters may be empty)
  };
  int pos = blockIdx.x >> 3;
  if (!locate(pos)) return;
  bool none;  // rows of no group
  int red, prows;
  const uint8_t *q0, *p0;
  const int64_t ldq = p.ldq * 2, ldp = p.ldp * 2;
  auto enter = [&] {
    none = !QA && e >= (p.counts ? p.groups : 1);
    red = QA ? nrows : none ? 0 : p.red;
    q0 = static_cast<const uint8_t*>(p.q) +
         (QA ? first * ldq + static_cast<int64_t>(rt) * T * 2 : first * ldq);
    p0 = static_cast<const uint8_t*>(p.p) + (QA ? first * ldp : e * p.p_group * 2) +
         (PA ? static_cast<int64_t>(ct) * T * 2 : static_cast<int64_t>(ct) * TN * ldp);
    if (none) p0 = static_cast<const uint8_t*>(p.p);
    prows = PA ? 0 : min(TN, p.n - ct * TN);
  };
  enter();
  // (a stage of zeros where there are no sums: the accumulators then come from the
  // loop alone, not from a choice that the compiler would make in VGPRs)
  auto stages = [&] { return max(1, (red + KB - 1) / KB); };

  // ---- the bias, where the accumulators start: its loads go out before the
  // stages'.
  constexpr int WN = 32 * NB;              // columns of a wave's accumulators
  constexpr int OC = GATED ? WN / 2 : WN;  // ... of its output
  int col0 = ct * TN + wn * OC;
  const int wide = GATED ? 2 * p.n : p.n;
  const int h = lane >> 5;
  uint2 bias[NB][4];
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      bias[j][g] = uint2{0, 0};
      const int c = col0 + (GATED ? j >> 1 : j) * 32 + 8 * g + 4 * h;
      if (FORWARD && p.bias && !none && c < p.n)
        __builtin_memcpy(&bias[j][g],
                         static_cast<const raw*>(p.bias) + static_cast<int64_t>(e) * wide + c +
                             (GATED && (j & 1) ? p.n : 0), 8);
    }

  // ---- operands. A stage's resource begins at the stage and ends with its last
  // value: `along`, with the tile's last row's last sum; `across`, with the last
  // row's last column (rows lie at least their width apart: check_linear_across).
  Feed<C, QA> fq;
  Feed<C, PA> fp;
  // (gated: the tile's rows of P by 32: gate, up, gate, up ... of the same columns; the
  // up rows' resource starts n rows further on)
  fq.init(wave, lane, ldq, [](int r) { return r; });
  fp.init(wave, lane, ldp, [](int r) { return GATED ? (r >> 6) * 32 + (r & 31) : r; });
  // `bytes` of them, none unless left > 0. (By a mask: with a branch, which the
  // compiler makes of a choice here, a stage's instructions cannot be ordered: the
  // products stood still for the LDS reads, 8 % more time.)
  auto resource = [](const uint8_t* base, int bytes, int left) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0,
                                             bytes & ~((left - 1) >> 31), kBufWord3);
  };
  auto feed = [&](auto across_c, const auto& f, const uint8_t* base, int64_t ld, int rows,
                  int width, int s, uint8_t* dst, bool up) {
    constexpr bool ACROSS = decltype(across_c)::value;
    const int ld32 = static_cast<int>(ld);
    if constexpr (ACROSS) {
      const int left = red - s * KB;
      const __amdgpu_buffer_rsrc_t r =
          resource(base + static_cast<int64_t>(s) * KB * ld,
                   (min(KB, left) - 1) * ld32 + width * 2, left);
#pragma unroll
      for (int i = 0; i < NL; ++i) lds_dma16_buf(r, f.off[i], 0, dst + i * 1024);
    } else {
      const int left = (red - s * KB) * 2;  // bytes of sums from here on
      const uint8_t* b = base + static_cast<int64_t>(s) * (KB * 2);
      const int bytes = (rows - 1) * ld32 + left;
      const __amdgpu_buffer_rsrc_t r = resource(b, bytes, left);
      const __amdgpu_buffer_rsrc_t ru = resource(up ? b + p.n * ld : b, bytes, left);
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const bool is_up = up && (((wave * NL + i) * (512 / KB) >> 5) & 1);
        const uint32_t o = (f.c0 ^ ((i & 1) * f.FLIP)) < left ? f.off[i] : kOutside;
        if (is_up) lds_dma16_buf(ru, o, 0, dst + i * 1024);
        else lds_dma16_buf(r, o, 0, dst + i * 1024);
      }
    }
  };
  auto feed_q = [&](int s, int slot) {
    feed(std::integral_constant<bool, QA>{}, fq, q0, ldq, nrows, p.m - rt * T, s,
         lds + slot + wave * NL * 1024, false);
  };
  auto feed_p = [&](int s, int slot) {
    feed(std::integral_constant<bool, PA>{}, fp, p0, ldp, prows, p.n - ct * T, s,
         lds + P_AT + slot + wave * NL * 1024, GATED);
  };

  // ---- fragments: 32 rows x 16 sums, eight sums a lane. Q's blocks of a wave are
  // the tile's blocks 2i + wm, so that both halves share a short tile's rows.
  int along[C::KK];  // by 16 sums
#pragma unroll
  for (int kk = 0; kk < C::KK; ++kk)
    along[kk] = (lane & 31) * (KB * 2) + C::chunk(lane & 31, 2 * kk + h) * 16;
  int across[4];  // by block % 4: lane's row and 8 bytes
  const int a4 = (lane >> 2) & 3;
#pragma unroll
  for (int b = 0; b < 4; ++b)
    across[b] = (8 * h + a4) * (2 * T) + (b ^ a4) * 64 + ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
  auto read = [&](auto across_c, int slot, int block, int kk) -> Frag {
    if constexpr (decltype(across_c)::value) {
      const uint8_t* a = lds + slot + across[block & 3] + (block >> 2) * 256 + kk * 16 * 2 * T;
      const s16x4 lo = read_transposed((LdsWords)(a));
      const s16x4 hi = read_transposed((LdsWords)(a + 4 * 2 * T));
      return __builtin_bit_cast(Frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      return *reinterpret_cast<const Frag*>(lds + slot + block * 32 * KB * 2 + along[kk]);
    }
  };
  f32x16 acc[NB][NB];
  Frag fa[2][NB], fb[2][NB];
  auto read_frags = [&](int oq, int op, int kk, Frag (&a)[NB], Frag (&b)[NB]) {
#pragma unroll
    for (int i = 0; i < NB; ++i)
      a[i] = read(std::integral_constant<bool, QA>{}, oq, 2 * i + wm, kk);
#pragma unroll
    for (int j = 0; j < NB; ++j)
      b[j] = read(std::integral_constant<bool, PA>{}, P_AT + op, wn * NB + j, kk);
  };
  auto mma = [&](const Frag (&a)[NB], const Frag (&b)[NB]) {
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[i][j] = M::mma32(b[j], a[i], acc[i][j]);
  };

  // The order of a step's instructions: the next step's LDS reads behind the first
  // MFMAs, then the loads (0 or NL) spread over the others.
  constexpr int NM = NB * NB, NR = NB * ((QA ? 2 : 1) + (PA ? 2 : 1));
  auto order = [&](auto loads_c) {
    constexpr int LOADS = decltype(loads_c)::value;
    // MFMAs for the reads
    constexpr int MR = LOADS > 0 && NM - LOADS > NM / 2 ? NM - LOADS : NM / 2;
    constexpr int PER = (NR + MR - 1) / MR, RM = (NR + PER - 1) / PER;
    constexpr int LPM = LOADS ? (LOADS + NM - RM - 1) / (NM - RM) : 1;
    static_for<RM>([&](auto) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);
    });
    static_for<(LOADS + LPM - 1) / LPM>([&](auto) {
      __builtin_amdgcn_sched_group_barrier(0x020, LPM, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    });
  };

  // ---- main loop. Stage s lives in slot s % SLOTS of each ring. The barrier before its
  // last 16 sums publishes stage s + 1 (every wave has waited for its own loads of it)
  // and frees stage s's slots. P's loads of stage s + AHEAD go out during the first 16
  // sums, into the slot of stage s - 1; Q's after the barrier, into stage s - 1's
  // (five slots) or s's own (two).
  constexpr int AHEAD = KB == 32 ? 4 : 2;
  constexpr std::integral_constant<int, NL> loads{};
  constexpr std::integral_constant<int, 0> no_loads{};
  auto next_q = [](int o) { return o == (C::Q_SLOTS - 1) * SLOT ? 0 : o + SLOT; };
  auto next_p = [](int o) { return o == (C::P_SLOTS - 1) * SLOT ? 0 : o + SLOT; };
  // (ROUNDS: the first PRE stages of a tile go out before the epilogue of the one before)
  constexpr int PRE = ROUNDS ? 3 : AHEAD;
  constexpr int STORES = ROUNDS ? T * TN / (8 * 256) : 0;  // of a wave
#pragma unroll
  for (int s = 0; s < PRE; ++s) {
    feed_p(s, s * SLOT);
    feed_q(s, s * SLOT);
  }
  // (the first tile has no stores before it: the waits that leave room for them would be
  // too short)
  if constexpr (ROUNDS) wait_vmcnt<0>();
  for (;;) {
#pragma unroll
    for (int s = PRE; s < AHEAD; ++s) {
      feed_p(s, s * SLOT);
      feed_q(s, s * SLOT);
    }
    const int KT = stages();
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const uint32_t w = t < 2 ? bias[j][g].x : bias[j][g].y;
          const float v = FORWARD ? Elem<TY>::to_f32(static_cast<raw>(w >> (16 * (t & 1)))) : 0.f;
#pragma unroll
          for (int i = 0; i < NB; ++i) acc[i][j][4 * g + t] = v;
        }
    wait_vmcnt<2 * (AHEAD - 1) * NL + STORES>();
    wave_barrier_all();
    read_frags(0, 0, 0, fa[0], fb[0]);
    int oq = 0, op = 0, to_q = AHEAD % C::Q_SLOTS * SLOT, to_p = AHEAD % C::P_SLOTS * SLOT, s = 0;
    // MORE: vector memory operations that are in flight beside the loads
    auto stage = [&](auto more_c) {
      constexpr int MORE = decltype(more_c)::value;
#pragma unroll
      for (int kk = 0; kk + 1 < C::KK; ++kk) {
        read_frags(oq, op, kk + 1, fa[(kk + 1) & 1], fb[(kk + 1) & 1]);
        if (kk == 0) feed_p(s + AHEAD, to_p);
        mma(fa[kk & 1], fb[kk & 1]);
        if (kk == 0) order(loads);
        else order(no_loads);
        __builtin_amdgcn_sched_barrier(0);
      }
      wait_lgkm0();
      // behind stage s + 1's loads: those of the stages to s + AHEAD - 1, and P's
      wait_vmcnt<(2 * (AHEAD - 2) + 1) * NL + MORE>();
      wave_barrier_all();
      __builtin_amdgcn_sched_barrier(0);
      oq = next_q(oq);
      op = next_p(op);
      read_frags(oq, op, 0, fa[0], fb[0]);
      feed_q(s + AHEAD, to_q);
      to_q = next_q(to_q);
      to_p = next_p(to_p);
      mma(fa[1], fb[1]);
      order(loads);
      __builtin_amdgcn_sched_barrier(0);
    };
    // (the loads of the first PRE stages are older than the stores of the tile before)
    if constexpr (ROUNDS) {
      const int n = min(KT, PRE - 1);
      do stage(std::integral_constant<int, STORES>{});
      while (++s < n);
    }
    if (!ROUNDS || s < KT) {
      do stage(std::integral_constant<int, 0>{});
      while (++s < KT);
    }
    wait_vmcnt<0>();
    wait_lgkm0();
    wave_barrier_all();  // the ring is done with

    // ---- epilogue. Activation and residual are taken in fp32 in the accumulators'
    // layout (a gate and its up value are two registers of a lane), then
    // rounded; the wave's whole part goes through LDS in 16 bits so that it leaves as
    // runs of a row, 16 bytes a lane. The residual comes in the same way first; z, which
    // a gradient is taken at, leaves in fp32 (in 16 bits, its rounding was as large a
    // part of the gradients' error as their own).
    uint8_t* stg = lds + (ROUNDS ? (wave >> 1) * P_AT + PRE * SLOT + (wave & 1) * SLOT
                                 : wave * C::STAGING);
    // (the weights' gradient: rows of the group's matrix)
    const int64_t row0 = QA ? static_cast<int64_t>(e) * p.m + rt * T : first;
    const int rows_in = QA ? min(T, p.m - rt * T) : nrows;
    bool more = false;
    const int out0 = col0;
    if constexpr (ROUNDS) {
      pos += 32;
      more = locate(pos);
      if (more) {
        enter();
        col0 = ct * TN + wn * OC;
#pragma unroll
        for (int s = 0; s < PRE; ++s) {
          feed_p(s, s * SLOT);
          feed_q(s, s * SLOT);
        }
      }
    }
    // Eight bytes s of staged row r: the XOR spreads a column of 32 rows over all banks.
    // Sixteen bytes are two of them, swapped in some rows.
    constexpr int W8 = OC / 4, RPL = 32 / W8;
    auto place = [](int r, int s) { return r * W8 * 8 + (s ^ ((r / RPL) & (W8 - 1))) * 8; };
    auto sync = [] {
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };
    // Both of (staged row, output row in the tile, 16-byte chunk, k) for the wave's part,
    // a chunk a lane, k of up to eight at a time; the tile's rows 64 i + 32 wm + r are the staged
    // rows 32 i + r.
    constexpr int PARTS = ROUNDS ? 2 : 1, PB = NB / PARTS;
    auto runs = [&](auto&& get, auto&& put) {
      constexpr int LPR = OC / 8, RPP = 64 / LPR;
      constexpr int RUNS = WN / PARTS / RPP, AT = RUNS < 8 ? RUNS : 8;
      static_assert(RUNS % AT == 0, "runs");
      const int lr = lane / LPR, lc = lane % LPR;
      for (int k0 = 0; k0 < RUNS; k0 += AT) {
#pragma unroll
        for (int k = 0; k < AT; ++k) {
          const int sr = (k0 + k) * RPP + lr;
          get(sr, (sr >> 5) * 64 + wm * 32 + (sr & 31), lc, k);
        }
#pragma unroll
        for (int k = 0; k < AT; ++k) {
          const int sr = (k0 + k) * RPP + lr;
          put(sr, (sr >> 5) * 64 + wm * 32 + (sr & 31), lc, k);
        }
      }
    };
    auto pack4 = [](const float (&v)[4]) {
      return uint2{pack2<TY>(v[0], v[1]), pack2<TY>(v[2], v[3])};
    };
    // (Accumulators stay where they are until they are used: otherwise the compiler
    // reads all of them into VGPRs ahead, more than there are.)
    auto keep = [](f32x16& a) { asm volatile("" : "+a"(a)); };
    const int r32 = lane & 31;
    if (FORWARD && p.z) {
      // in fp32, 32 rows at a time: chunks of four values, spread over the banks
      constexpr int CH = WN / 4, RPP = 64 / CH;
      auto chunk = [&](int r, int c) {
        return reinterpret_cast<f32x4*>(stg + (r * CH + ((c ^ (r & 15)) & (CH - 1))) * 16);
      };
      const int lc = lane % CH;
      const int zc = col0 + (GATED ? (lc >> 4) * 32 : (lc >> 3) * 32) + (lc & 7) * 4;
      const int64_t to = zc + (GATED && ((lc >> 3) & 1) ? p.n : 0);
      static_for<NB>([&](auto i_c) {
        constexpr int i = decltype(i_c)::value;
#pragma unroll
        for (int j = 0; j < NB; ++j) {
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *chunk(r32, j * 8 + 2 * g + h) = f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1],
                                                   acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
        }
        sync();
#pragma unroll
        for (int k = 0; k < 32 / RPP; ++k) {
          const int sr = k * RPP + lane / CH, r = i * 64 + wm * 32 + sr;
          const f32x4 v = *chunk(sr, lc);
          if (r < rows_in && zc < p.n)
            *reinterpret_cast<f32x4*>(p.z + (row0 + r) * wide + to) = v;
        }
        sync();
      });
    }
    if (FORWARD && p.residual) {
      u32x4 v[8];
      runs([&](int, int r, int c, int k) {
        v[k] = u32x4{0, 0, 0, 0};
        if (r < rows_in && col0 + c * 8 < p.n)
          v[k] = *reinterpret_cast<const u32x4*>(static_cast<const raw*>(p.residual) +
                                                 (row0 + r) * p.ldr + col0 + c * 8);
      }, [&](int sr, int, int c, int k) {
        if ((sr / RPL) & 1) v[k] = u32x4{v[k][2], v[k][3], v[k][0], v[k][1]};
        *reinterpret_cast<u32x4*>(stg + (place(sr, 2 * c) & ~15)) = v[k];
      });
      sync();
    }
    const bool has_residual = FORWARD && p.residual;
    // (rows of no group: sums of nothing, whose activations are 0)
    // (without a branch, so that every tile has STORES of them: what is outside is dropped)
    const __amdgpu_buffer_rsrc_t to = __builtin_amdgcn_make_buffer_rsrc(
        static_cast<raw*>(p.out) + row0 * p.n + out0, 0, 0x7fffffff, kBufWord3);
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
      const int I0 = part * PB;
#pragma unroll
      for (int i = I0; i < I0 + PB; ++i)
#pragma unroll
        for (int j = 0; j < NB; j += GATED ? 2 : 1) {
          auto at = [&](int g) {
            return reinterpret_cast<uint2*>(
                stg + place((i - I0) * 32 + r32, (GATED ? j >> 1 : j) * 8 + 2 * g + h));
          };
          keep(acc[i][j]);
          if constexpr (GATED) keep(acc[i][j + 1]);
          uint2 res[4];
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            res[g] = FORWARD ? *at(g) : uint2{0, 0};  // (without a residual: what the ring left)
            res[g].x = has_residual ? res[g].x : 0;
            res[g].y = has_residual ? res[g].y : 0;
          }
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            float v[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              v[t] = acc[i][j][4 * g + t];
              if constexpr (FORWARD) {
                v[t] = linear_act<ACT>(v[t]);
                if constexpr (GATED) v[t] *= acc[i][j + 1][4 * g + t];
                v[t] += Elem<TY>::to_f32(
                    static_cast<raw>((t < 2 ? res[g].x : res[g].y) >> (16 * (t & 1))));
              }
            }
            if constexpr (ROUNDS) put_staged(at(g), pack4(v));
            else *at(g) = pack4(v);
          }
        }
      sync();
      u32x4 v[8];  // (read together: one by one, each store waits for its read)
      runs([&](int sr, int, int c, int k) {
        const u32x4* from = reinterpret_cast<const u32x4*>(stg + (place(sr, 2 * c) & ~15));
        v[k] = ROUNDS ? staged(from) : *from;
      }, [&](int sr, int r, int c, int k) {
        if ((sr / RPL) & 1) v[k] = u32x4{v[k][2], v[k][3], v[k][0], v[k][1]};
        r += I0 * 64;
        const bool in = r < rows_in && out0 + c * 8 < p.n;
        __builtin_amdgcn_raw_buffer_store_b128(
            v[k], to, in ? static_cast<uint32_t>(r * p.n + c * 8) * 2 : kOutside, 0, 0);
      });
      if (PARTS > 1) sync();
    }
    if (!more) break;
    wait_lgkm0();
    wave_barrier_all();  // the staging is done with
  }
}

// ---------------------------------------------------------------- schedule ---
namespace {

template <int TY, int MODE, int ACT, int T>
int launch_tile(const LinearParams& p, int64_t wgs, hipStream_t stream) {
  typedef LinearTile<T, T == 256 && (MODE == kLinearDgrad || MODE == kLinearWgrad) ? 32 : 64> C;
  static std::atomic<uint64_t> told{0};
  return launch_lds("linear_tile_kernel", linear_tile_kernel<TY, MODE, ACT, C>, told,
                    C::ROUNDS ? std::min<int64_t>(wgs, 256) : wgs, 256, C::LDS, stream, p);
}
template <int TY, int MODE, int ACT>
int launch_form(const LinearParams& p, bool large, hipStream_t stream) {
  const int t = large ? 256 : 128, tn = MODE == kLinearGated ? t / 2 : t;
  const int64_t nc = (p.n + tn - 1) / tn;
  const int64_t nr = MODE == kLinearWgrad ? static_cast<int64_t>(p.groups) * ((p.m + t - 1) / t)
                                          : linear_row_tiles(p, t);
  const int64_t tiles = nr * nc;
  if (tiles > 0x7fffffffll) return fail(FGS_EUNSUPPORTED, "too many tiles for a grid");
  if (const int rc = check_linear_across(p, MODE)) return rc;
  const int64_t wgs = (tiles + 7) / 8 * 8;
  if (!large) return launch_tile<TY, MODE, ACT, 128>(p, wgs, stream);
  // how many tiles there are is the device's to know where rows are grouped
  const bool known = MODE == kLinearWgrad || !p.counts;
  bool cut = !known && tiles > 256;
  if (known)
    for (int xcd = 0; xcd < 8; ++xcd)
      cut |= linear_rest(linear_share(static_cast<int>(tiles), xcd)) > 0;
  LinearParams q = p;
  q.part = cut ? kLinearCut : kLinearWhole;
  const int rc = launch_tile<TY, MODE, ACT, 256>(q, wgs, stream);
  if (rc || !cut) return rc;
  q.part = kLinearRest;
  return launch_tile<TY, MODE, ACT, 128>(q, 8 * 16 * 4, stream);
}
template <int TY>
int launch_type(const LinearParams& p, int mode, bool large, hipStream_t stream) {
  if (mode == kLinearDgrad) return launch_form<TY, kLinearDgrad, FGS_ACT_NONE>(p, large, stream);
  if (mode == kLinearWgrad) return launch_form<TY, kLinearWgrad, FGS_ACT_NONE>(p, large, stream);
  return with_act(p.act, [&](auto act_c) {
    constexpr int ACT = decltype(act_c)::value;
    return mode == kLinearGated ? launch_form<TY, kLinearGated, ACT>(p, large, stream)
                                : launch_form<TY, kLinearForward, ACT>(p, large, stream);
  });
}

}  // namespace

// The forms (FGS_LINEAR_FORM(i)): tile in rows x weight rows; blocks of 64 sums that an
// iteration takes (the streaming forms' waves take one each); workgroups that run at
// once; microseconds of an iteration, of one with half of them or fewer, beside the
// iterations of a round, and the TB/s at which the weights come: fitted to 590 products
// of 84 sizes, weights not in a cache (dense: 1 to 2048 rows, n 512 to 14336, k 512 to
// 7168; 8, 64 and 128 groups, 8 to 16384 rows). The choice takes 1.2 % more than the best
// form of each, 16 % at most.
// Measured at n and k 4096 (rows: us): 1: 8.1 (form 0; 36.6 in 128 x 128 tiles), 64: 12.6
// (2; 37.5), 128: 15.8 (3; 39.9), 256: 19.6 (4; 39.1), 512: 34.7 (4; 38.7), 1024: 41.2 (5; 79
// in 256 x 256), 2048: 67 (5; 85), 4096: 109 (6; 127).
struct LinearForm {
  int bm, bn, step, at_once;
  double iter, half, round, tbs;
  const char* name;
};
constexpr LinearForm kForms[] = {
    {16, 16, 8, 512, 0.93, 0.49, 0.74, 5.6, "stream 16x16"},
    {16, 32, 8, 256, 0.76, 0.73, 0.94, 5.4, "stream 16x32"},
    {32, 32, 8, 256, 1.14, 0.88, 0.87, 5.8, "stream 32x32"},
    {64, 32, 4, 256, 0.81, 0.66, 1.06, 8.0, "stream 64x32"},
    {64, 64, 4, 256, 1.10, 0.99, 1.66, 6.2, "stream 64x64"},
    {128, 128, 1, 512, 1.01, 0.57, 1.45, 5.6, "tiled 128x128"},
    {256, 256, 1, 256, 1.38, 1.08, 7.49, 8.0, "tiled 256x256"},
};
// The gradients', fitted in the same way: of the input, by the weights' columns (1 row at
// n and k 4096 18.7 us, 34.9 in 128 x 128 tiles; 128: 20.3 and 39.4; 512: 38.0 and 38.7;
// 68 sizes, 0.4 % more than the best on average), and of the weights (32 sizes).
constexpr LinearForm kInputForms[] = {
    {16, 64, 8, 256, 1.36, 1.78, 0.60, 5.2, "stream 16x64"},
    {32, 64, 4, 256, 0.87, 0.98, 0.88, 5.2, "stream 32x64"},
    {64, 64, 4, 256, 1.19, 1.17, 1.04, 5.6, "stream 64x64"},
    {128, 128, 1, 512, 1.07, 0.54, 0.67, 5.8, "tiled 128x128"},
    {256, 256, 1, 256, 1.35, 1.09, 4.65, 8.0, "tiled 256x256"},
};
constexpr LinearForm kWeightForms[] = {
    {128, 128, 1, 512, 0.98, 0.45, 2.39, 3.8, "tiled 128x128"},
    {256, 256, 1, 256, 1.50, 1.04, 6.48, 5.1, "tiled 256x256"},
};
struct LinearForms {
  const LinearForm* list;
  int count;  // the last two: tiles
};
LinearForms forms_of(int mode) {
  if (mode == kLinearDgrad) return {kInputForms, 5};
  if (mode == kLinearWgrad) return {kWeightForms, 2};
  return {kForms, 7};
}

bool linear_flags_ok(int mode, int32_t flags) {
  return flags >= 0 && flags <= forms_of(mode).count;
}

// The form with the shortest estimate. (Gated, the forward form 0 is form 1.)
int linear_form(int mode, int64_t groups, int64_t rows, int64_t m, int64_t n, int64_t red,
                int32_t flags) {
  if (flags) return flags - 1;
  const LinearForms forms = forms_of(mode);
  const double g = static_cast<double>(groups), r = static_cast<double>(rows);
  // groups with rows, if rows fall on them evenly; for the weights' gradient all have
  // an output
  const double used = groups > 1 ? g * -std::expm1(-r / g) : 1;
  const double wide = static_cast<double>(n) * (mode == kLinearGated ? 2 : 1);
  const double sums = mode == kLinearWgrad ? r / g : static_cast<double>(red);
  const double mb = mode == kLinearWgrad ? g * static_cast<double>(m) * wide * 2e-6
                                         : used * wide * sums * 2e-6;
  int best = forms.count - 1;
  double best_us = 0;
  for (int f = forms.count - 1; f >= (mode == kLinearGated ? 1 : 0); --f) {
    const LinearForm& q = forms.list[f];
    const double tall = mode == kLinearWgrad ? g * std::ceil(static_cast<double>(m) / q.bm)
                        : groups > 1         ? std::max(used, r / q.bm + used / 2)
                                             : std::ceil(r / q.bm);
    const double wgs = tall * std::ceil(wide / q.bn);
    const double iters = std::ceil(std::ceil(sums / 64) / q.step);
    const double iter = wgs <= q.at_once / 2 ? q.half : q.iter;
    const double look = groups > 1 ? 0.7 * std::ceil(g / 64) : 0;  // for a tile's group
    const double round = iters * iter + q.round + look;
    double rounds = std::ceil(wgs / q.at_once);
    if (q.bm == 256) {  // (a last round that is cut off: its quarters')
      const double rest = wgs / q.at_once - std::floor(wgs / q.at_once);
      if (wgs > q.at_once && rest > 0 && rest <= 0.5) rounds += (rest <= 0.25 ? 0.45 : 0.75) - 1;
    }
    // (the gradients' workgroups load ahead and store behind from tile to tile)
    const double saved = q.bm < 256 ? 0 : mode == kLinearWgrad ? 3 : mode == kLinearDgrad ? 2 : 0;
    const double c = rounds * round - saved * std::max(0.0, rounds - 1);
    const double w = mb / q.tbs;
    const double us = c * c * c * c + w * w * w * w;  // (of the two, the longer one counts)
    if (f == forms.count - 1 || us < best_us) {
      best = f;
      best_us = us;
    }
  }
  return best;
}

std::string linear_form_name(int mode, int form) {
  return forms_of(mode).list[mode == kLinearGated && form == 0 ? 1 : form].name;
}

int launch_linear(const LinearParams& p, int mode, int dtype, int form, hipStream_t stream) {
  const int tiles = forms_of(mode).count - 2;
  if (form < tiles) return launch_linear_small(p, mode, dtype, form, stream);
  const bool large = form > tiles;
  return dtype == FGS_DTYPE_BF16 ? launch_type<FGS_DTYPE_BF16>(p, mode, large, stream)
                                 : launch_type<FGS_DTYPE_FP16>(p, mode, large, stream);
}

}  // namespace fgs

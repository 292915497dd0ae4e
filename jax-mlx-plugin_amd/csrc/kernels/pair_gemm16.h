// Products of matrices held as sums of two 16-bit terms, leading and second ones
// (newton_schulz.hip):
//
//   C[m][n] = sum_k A_lo B_hi + A_hi B_hi + A_hi B_lo        fp32 accumulation
//
// (A_lo B_lo lies below what the two terms of either operand leave out.)  Tiles,
// wavefronts and operand forms are those of xent_gemm16.h; each tile of 16 k
// brings both terms of both operands, so that three products of a block share
// its reads: a step of each, in the order above, needs one new set of fragments at
// a time, and 32 reads and 8 loads a wavefront feed 96 products of a 128 x 128
// block, where three walks along k would take 48 and 24.
//
// Schedule of 128 x 128 and 64 x 64 blocks.  Four LDS stages, loaded three tiles ahead.  Step 0 multiplies A_lo by
// B_hi and reads A_hi, step 1 A_hi by B_hi and reads B_lo, and the loads of the
// tile three ahead go out between the products of both; step 2 multiplies A_hi by B_lo,
// and at its slot B0 the next tile has landed for everyone (the one barrier of a
// tile) and its A_lo and B_hi are read.
#pragma once

#include "xent_gemm16.h"

namespace mfx {
namespace xent {

// Chunk c of a k-contiguous tile's row r (32 bytes, or 64 of 32 k) at c ^
// pair_swz(r): the 16 rows that a 16-byte read serves at a time spread over all
// banks.
template <int BK>
__device__ __forceinline__ int pair_swz(int r) {
  return BK == 16 ? (r >> 3) & 1 : kc_swz(r);
}

// One operand's tiles of BK k, leading terms and behind them second ones (TERM
// elements each).  KC: [IDX rows][BK], else [BK][IDX], chunk c of row r at c ^
// tile_swz.
template <bool KC, int IDX, int NW, int BK>
struct PairTile {
  static constexpr int TERM = IDX * BK;
  static constexpr int RPI = KC ? 512 / BK : 512 / IDX;  // rows one load instruction covers
  static constexpr int ROWS = KC ? IDX : BK;
  static constexpr int LOADS = ROWS / (RPI * NW);  // of a term
  static_assert(LOADS >= 1 && LOADS * RPI * NW == ROWS, "whole loads");
  static constexpr int STEP = RPI * NW;
  static_assert(STEP % 16 == 0 || (!KC && STEP == 8), "one or two source chunks per lane");
  static constexpr int NOFF = STEP % 16 == 0 ? 1 : 2;

  const bf16* cur;      // the next tile's first leading term
  int64_t next, lo;     // elements from tile to tile, and to the second terms
  int k0, K, left;      // the next tile's first k; tiles left
  int ld2, last;        // as in Tile
  uint32_t voff[NOFF], vo;
  int lane_k;
#if defined(__HIP_DEVICE_COMPILE__)
  __amdgpu_buffer_rsrc_t hi, second;
#endif

  __device__ __forceinline__ PairTile(const Operand& o, int idx0, int total, int k, int kt0, int kt1, int wave, int lane) {
    const int rows = total - idx0;
    K = k;
    k0 = kt0 * BK;
    left = kt1 - kt0;
    ld2 = (int)o.ld * 2;
    lo = o.lo;
    next = KC ? BK : BK * o.ld;
    cur = static_cast<const bf16*>(o.p) + (KC ? (int64_t)idx0 * o.ld + k0 : (int64_t)k0 * o.ld + idx0);
    const int K8 = (K + 7) & ~7, rows8 = (rows + 7) & ~7;
    last = KC ? (min(rows, IDX) - 1) * ld2 + K8 * 2 : rows8 * 2;
    constexpr int CPR = KC ? BK / 8 : IDX / 8;
    const int row = wave * RPI + lane / CPR, slot = lane % CPR;
    const int chunk = KC ? slot ^ pair_swz<BK>(row) : slot ^ tile_swz<IDX>(row);
    lane_k = chunk * 8;
#pragma unroll
    for (int i = 0; i < NOFF; ++i) voff[i] = (uint32_t)(row * ld2 + (chunk ^ (i * 8)) * 16);
    vo = voff[0];
  }
  // Takes up the next tile: its resources (empty past the last).
  __device__ __forceinline__ void take() {
#if defined(__HIP_DEVICE_COMPILE__)
    int extent = KC ? last - k0 * 2 : (min(K - k0, BK) - 1) * ld2 + last;
    if (left-- <= 0) extent = 0;
    hi = __builtin_amdgcn_make_buffer_rsrc(const_cast<bf16*>(cur), (short)0, extent, 0x00020000);
    second = __builtin_amdgcn_make_buffer_rsrc(const_cast<bf16*>(cur + lo), (short)0, extent, 0x00020000);
    if constexpr (KC) vo = k0 + lane_k < K ? voff[0] : kOOR;
    cur += next;
    k0 += BK;
#endif
  }
  // Load l of 2 * LOADS: the leading terms' first.
  __device__ __forceinline__ void load(int l, bf16* lds, int wave) const {
#if defined(__HIP_DEVICE_COMPILE__)
    const int i = l % LOADS;
    const uint32_t v = (NOFF == 1 ? vo : voff[i % NOFF]) + (uint32_t)(i * STEP * ld2);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(l < LOADS ? hi : second,
                                             (tiles::lds_void_t*)(lds + (l / LOADS) * TERM + (NW * i + wave) * 64 * 8),
                                             16, v, 0, 0, 0);
#endif
  }
};

// Fragments of NB neighbouring 32-index blocks (Frag, xent_gemm16.h) of the KS-th
// 16 k of a tile.
template <bool KC, int IDX, int NB, int BK>
struct PairReader {
  static constexpr int NA = KC ? BK / 16 : 2 * NB;
  static constexpr int READS = KC ? NB : 2 * NB;
  static constexpr int TERM = IDX * BK * 2;  // bytes
  uint32_t a[NA];
  __device__ __forceinline__ PairReader(uint32_t tile, int blk0, int lane) {
    const int half = lane >> 5, l32 = lane & 31;
    if constexpr (KC) {
#pragma unroll
      for (int ks = 0; ks < NA; ++ks)
        a[ks] = tile + (uint32_t)((blk0 * 32 + l32) * BK * 2 + ((2 * ks + half) ^ pair_swz<BK>(l32)) * 16);
    } else {
      const int tj = lane & 15, tg = (lane >> 4) & 1;
      const int r = 8 * half + (tj >> 2);
      const int chunk = tg * 2 + ((tj & 3) >> 1), sub = (tj & 1) * 8;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int c = (blk0 + b) * 4 + chunk;
        a[2 * b] = tile + (uint32_t)(r * IDX * 2 + (c ^ tile_swz<IDX>(r)) * 16 + sub);
        a[2 * b + 1] = tile + (uint32_t)((r + 4) * IDX * 2 + (c ^ tile_swz<IDX>(r + 4)) * 16 + sub);
      }
    }
  }
  // Read R of the leading (LO 0) or second terms.
  template <int KS, int LO, int R>
  __device__ __forceinline__ void read(Frag<KC> (&f)[NB]) const {
    constexpr int STEP = KS * 16 * IDX * 2;  // (index-contiguous: rows are k; whole swizzle periods)
    if constexpr (KC) tiles::ds_b128<LO * TERM + R * 32 * BK * 2>(f[R].v, a[KS]);
    else if constexpr (R & 1) tiles::ds_tr<LO * TERM + STEP>(f[R / 2].hi, a[R]);
    else tiles::ds_tr<LO * TERM + STEP>(f[R / 2].lo, a[R]);
  }
  __device__ __forceinline__ void move(uint32_t by) {
#pragma unroll
    for (int i = 0; i < NA; ++i) a[i] += by;
  }
};

// The sums of tile (m0, n0) over the tiles [kt0, kt1) of 16 k (at least one).
// smem: C::STAGES (a power of two) stages of 2 (BM + BN) 16 elements.  Tiles past
// the last are loaded out of range, as zeros, so that the loads in flight, which
// the waits count, do not depend on the tile.
template <class C>
__device__ __forceinline__ void gemm_pair16(const GemmShape& g, int m0, int n0, int kt0, int kt1, bf16* smem,
                                            Acc<C>& acc) {
  constexpr int FM = C::FM, FN = C::FN, NQ = FM * FN;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % C::WM, wn = wave / C::WM;
  using TA = PairTile<C::A_KC, C::BM, C::NW, 16>;
  using TB = PairTile<C::B_KC, C::BN, C::NW, 16>;
  constexpr int LA = 2 * TA::LOADS, NL = LA + 2 * TB::LOADS;
  constexpr int STAGE = 2 * (TA::TERM + TB::TERM) * 2;  // bytes
  constexpr int NS = C::STAGES, AHEAD = (NS - 2) * NL;  // loads in flight behind those of the next tile
  static_assert(NS * STAGE <= C::SMEM && AHEAD < 64, "the stages; the counter's range");
  TA ta(g.a, m0, g.M, g.K, kt0, kt1, wave, lane);
  TB tb(g.b, n0, g.N, g.K, kt0, kt1, wave, lane);
  const uint32_t lds = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)smem;
  using RA = PairReader<C::A_KC, C::BM, FM, 16>;
  using RB = PairReader<C::B_KC, C::BN, FN, 16>;
  RA ra(lds, wm * FM, lane);
  RB rb(lds + 2 * TA::TERM * 2, wn * FN, lane);
  constexpr int NRA = RA::READS, NRB = RB::READS;

#pragma unroll
  for (int j = 0; j < FN; ++j)
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[j][i][e] = 0.f;

  Frag<C::A_KC> fa[2][FM];  // leading, second terms
  Frag<C::B_KC> fb[2][FN];
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  // The named fragments have landed: their uses come after this.
  auto landed = [&](auto a_tag, auto b_tag) __attribute__((always_inline)) {
    constexpr int A = decltype(a_tag)::value, B = decltype(b_tag)::value;  // (2: none of them)
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if constexpr (A < 2)
#pragma unroll
      for (int i = 0; i < FM; ++i) fa[A][i].tie();
    if constexpr (B < 2)
#pragma unroll
      for (int j = 0; j < FN; ++j) fb[B][j].tie();
    fence();
  };
  using None = std::integral_constant<int, 2>;
  auto read_a = [&](auto lo_tag, auto r_tag) __attribute__((always_inline)) {
    constexpr int LO = decltype(lo_tag)::value, r = decltype(r_tag)::value;
    ra.template read<0, LO, r>(fa[LO]);
  };
  auto read_b = [&](auto lo_tag, auto r_tag) __attribute__((always_inline)) {
    constexpr int LO = decltype(lo_tag)::value, r = decltype(r_tag)::value;
    rb.template read<0, LO, r>(fb[LO]);
  };
  // The products of A's terms SA and B's SB in order, with between(q) ahead of product q.
  auto multiply = [&](auto a_tag, auto b_tag, auto between) __attribute__((always_inline)) {
    constexpr int A = decltype(a_tag)::value, B = decltype(b_tag)::value;
    tiles::static_for<0, NQ>([&](auto q_tag) {
      constexpr int q = decltype(q_tag)::value, j = q / FM, i = q % FM;
      between(q_tag);
      fence();
      acc[j][i] = mfma16<C::E>(fb[B][j].bits(), fa[A][i].bits(), acc[j][i]);
      fence();
    });
  };
  // Of N things spread over the slots [A, B), those of slot q.
  auto spread = [](auto q_tag, auto a_tag, auto b_tag, auto n_tag, auto f) __attribute__((always_inline)) {
    constexpr int q = decltype(q_tag)::value, a = decltype(a_tag)::value, b = decltype(b_tag)::value;
    constexpr int n = decltype(n_tag)::value;
    if constexpr (q >= a && q < b) tiles::static_for<(q - a) * n / (b - a), (q - a + 1) * n / (b - a)>(f);
  };
  auto load = [&](int l, bf16* to) __attribute__((always_inline)) {
    if (l < LA) ta.load(l, to, wave);
    else tb.load(l - LA, to + 2 * TA::TERM, wave);
  };
  constexpr int B0 = NQ >= 16 ? NQ / 4 : NQ / 2;  // the slot of step 2 with the barrier
  using Zero = I0;
  using Half = std::integral_constant<int, NQ / 2>;
  using Barrier = std::integral_constant<int, B0>;
  using Most = std::integral_constant<int, B0 + NQ / 2>;
  using NA = std::integral_constant<int, NRA>;
  using NB = std::integral_constant<int, NRB>;
  using NAB = std::integral_constant<int, NRA + NRB>;
  auto stage = [&](uint32_t s) { return smem + s * (STAGE / 2); };

  for (int t = 0; t < NS - 1; ++t) {
    ta.take();
    tb.take();
#pragma unroll
    for (int l = 0; l < NL; ++l) load(l, stage(t));
  }
  ta.take();
  tb.take();
  wait_loads<AHEAD>();
  barrier();
  tiles::static_for<0, NRA>([&](auto r) { read_a(I1{}, r); });
  tiles::static_for<0, NRB>([&](auto r) { read_b(I0{}, r); });
  landed(I1{}, I0{});
  uint32_t to = NS - 1;  // the stage being loaded
  for (int kt = kt0; kt < kt1; ++kt) {
    bf16* const fresh = stage(to);
    multiply(I1{}, I0{}, [&](auto q_tag) __attribute__((always_inline)) {
      constexpr int q = decltype(q_tag)::value;
      spread(q_tag, Zero{}, Half{}, NA{}, [&](auto r) { read_a(I0{}, r); });
#pragma unroll
      for (int l = q * NL / (2 * NQ); l < (q + 1) * NL / (2 * NQ); ++l) load(l, fresh);
    });
    landed(I0{}, None{});
    multiply(I0{}, I0{}, [&](auto q_tag) __attribute__((always_inline)) {
      constexpr int q = decltype(q_tag)::value;
      spread(q_tag, Zero{}, Half{}, NB{}, [&](auto r) { read_b(I1{}, r); });
#pragma unroll
      for (int l = (q + NQ) * NL / (2 * NQ); l < (q + NQ + 1) * NL / (2 * NQ); ++l) load(l, fresh);
    });
    landed(None{}, I1{});
    // (This tile's reads are done; the next stage, behind the last tile an empty
    // one's zeros, is read behind the barrier.)
    to = (to + 1) & (NS - 1);
    const uint32_t by = to == NS - 1 ? (uint32_t)(-(NS - 1) * STAGE) : (uint32_t)STAGE;
    multiply(I0{}, I1{}, [&](auto q_tag) __attribute__((always_inline)) {
      constexpr int q = decltype(q_tag)::value;
      if constexpr (q == 0) {
        ra.move(by);
        ta.take();
      }
      if constexpr (q == (NQ >= 4 ? 1 : 0)) {
        rb.move(by);
        tb.take();
      }
      if constexpr (q == B0) {
        wait_loads<AHEAD>();
        barrier();
      }
      spread(q_tag, Barrier{}, Most{}, NAB{}, [&](auto r) {
        constexpr int R = decltype(r)::value;
        if constexpr (R < NRA) read_a(I1{}, r);
        else read_b(I0{}, std::integral_constant<int, R - NRA>{});
      });
    });
    landed(I1{}, I0{});
  }
  wait_loads<0>();  // (those out of range: the stages are the caller's now)
}

// The same over tiles of 32 k, all of whose fragments are in registers before its products
// start and the next tile's are read beside them: for 64 x 64 blocks, of few products, and 96 x 96 of
// a wavefront, whose 54 cover taking up the next tile from two stages.
template <class C>
__device__ __forceinline__ void gemm_pair16_flat(const GemmShape& g, int m0, int n0, int kt0, int kt1, bf16* smem,
                                                 Acc<C>& acc) {
  constexpr int FM = C::FM, FN = C::FN, BK = 32, KS = BK / 16, PER = 3 * FM * FN, NQ = KS * PER;  // products of a tile
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % C::WM, wn = wave / C::WM;
  using TA = PairTile<C::A_KC, C::BM, C::NW, BK>;
  using TB = PairTile<C::B_KC, C::BN, C::NW, BK>;
  constexpr int LA = 2 * TA::LOADS, NL = LA + 2 * TB::LOADS;
  constexpr int STAGE = 2 * (TA::TERM + TB::TERM) * 2;
  constexpr int NS = C::STAGES, AHEAD = (NS - 2) * NL;
  static_assert(NS * STAGE <= C::SMEM && AHEAD + NL < 64, "the stages; the counter's range");
  TA ta(g.a, m0, g.M, g.K, kt0, kt1, wave, lane);
  TB tb(g.b, n0, g.N, g.K, kt0, kt1, wave, lane);
  const uint32_t lds = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)smem;
  using RA = PairReader<C::A_KC, C::BM, FM, BK>;
  using RB = PairReader<C::B_KC, C::BN, FN, BK>;
  RA ra(lds, wm * FM, lane);
  RB rb(lds + 2 * TA::TERM * 2, wn * FN, lane);
  constexpr int NRA = RA::READS, NRB = RB::READS, ONE = 2 * (NRA + NRB), NR = KS * ONE;

#pragma unroll
  for (int j = 0; j < FN; ++j)
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[j][i][e] = 0.f;

  struct Set {
    Frag<C::A_KC> a[KS][2][FM];  // leading, second terms
    Frag<C::B_KC> b[KS][2][FN];
  };
  Set set[2];
  // Read r of a tile: A_lo, B_hi, A_hi, B_lo.
  auto read = [&](Set& s, auto r_tag) __attribute__((always_inline)) {
    constexpr int ks = decltype(r_tag)::value / ONE, r = decltype(r_tag)::value % ONE;
    if constexpr (r < NRA) ra.template read<ks, 1, r>(s.a[ks][1]);
    else if constexpr (r < NRA + NRB) rb.template read<ks, 0, r - NRA>(s.b[ks][0]);
    else if constexpr (r < 2 * NRA + NRB) ra.template read<ks, 0, r - NRA - NRB>(s.a[ks][0]);
    else rb.template read<ks, 1, r - 2 * NRA - NRB>(s.b[ks][1]);
  };
  auto landed = [&](Set& s) __attribute__((always_inline)) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int t = 0; t < 2 * KS; ++t) {
#pragma unroll
      for (int i = 0; i < FM; ++i) s.a[t / 2][t % 2][i].tie();
#pragma unroll
      for (int j = 0; j < FN; ++j) s.b[t / 2][t % 2][j].tie();
    }
    fence();
  };
  auto load = [&](int l, bf16* to) __attribute__((always_inline)) {
    if (l < LA) ta.load(l, to, wave);
    else tb.load(l - LA, to + 2 * TA::TERM, wave);
  };
  for (int t = 0; t < NS; ++t) {
    ta.take();
    tb.take();
#pragma unroll
    for (int l = 0; l < NL; ++l) load(l, smem + t * (STAGE / 2));
  }
  wait_loads<AHEAD + NL>();
  barrier();
  tiles::static_for<0, NR>([&](auto r) { read(set[0], r); });
  landed(set[0]);
  uint32_t at = 0;  // the stage that the set in use came from: read, and loaded again
  // Multiplies set `now` of tile kt and reads the next tile's into the other.
  auto tile = [&](Set& now, Set& next) __attribute__((always_inline)) {
    bf16* const fresh = smem + at * (STAGE / 2);
    const uint32_t by = at == NS - 1 ? (uint32_t)(-(NS - 1) * STAGE) : (uint32_t)STAGE;
    at = (at + 1) & (NS - 1);
    ra.move(by);
    rb.move(by);
    ta.take();
    tb.take();
    wait_loads<AHEAD>();
    barrier();
    tiles::static_for<0, NQ>([&](auto q_tag) {
      constexpr int q = decltype(q_tag)::value, ks = q / PER, step = q % PER / (FM * FN);
      constexpr int j = q % (FM * FN) / FM, i = q % FM;
      constexpr int H = NQ / 2;  // (reads in the first half)
      if constexpr (q < H)
        tiles::static_for<q * NR / H, (q + 1) * NR / H>([&](auto r) __attribute__((always_inline)) { read(next, r); });
#pragma unroll
      for (int l = q * NL / NQ; l < (q + 1) * NL / NQ; ++l) load(l, fresh);
      fence();
      constexpr int A = step == 0 ? 1 : 0, B = step == 2 ? 1 : 0;
      acc[j][i] = mfma16<C::E>(now.b[ks][B][j].bits(), now.a[ks][A][i].bits(), acc[j][i]);
      fence();
    });
    landed(next);
  };
  int kt = kt0;
  for (; kt + 1 < kt1; kt += 2) {
    tile(set[0], set[1]);
    tile(set[1], set[0]);
  }
  if (kt < kt1) tile(set[0], set[1]);  // (what it reads are an empty tile's zeros)
  wait_loads<0>();
}

}  // namespace xent
}  // namespace mfx

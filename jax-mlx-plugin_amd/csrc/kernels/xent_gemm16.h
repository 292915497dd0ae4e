// The 16-bit product kernel of the linear cross entropy (linear_xent.hip) and
// of the Newton-Schulz iteration (newton_schulz.hip):
//
//   C[m][n] = sum_k A(m, k) B(n, k)        fp32 accumulation
//
// Each operand is stored either k-contiguous, [index][k], or index-contiguous,
// [k][index]; what happens to a tile's sums is the epilogue's business (a
// softmax's partial sums, a gradient, a store).  As in gemm16.hip the kernel
// computes C^T on v_mfma_f32_32x32x16 (its A operand taken from B): an
// accumulator lane then holds one row m and 16 columns n, so a row's maximum
// and sum need one exchange between two lanes.
//
// Tiles of 256 x 256 outputs by 4 wavefronts of 128 x 128 (one a SIMD, the sums
// in its 256 accumulation registers): 8 operand reads feed 16 products, half of
// what 64 x 64 a wavefront needs.  k advances by 32 through four LDS stages
// of 32 KB filled by LDS-DMA three tiles ahead.
//
// Schedule.  With one wavefront a SIMD nothing hides a stall, so every
// instruction that is not a product goes between two products, which occupy the
// matrix core for 32 cycles each: the operand reads of the next 16 k between
// the first products of a step, a tile's 8 loads one to two products (a CU takes
// their requests at about 90 bytes a cycle; together they would wait for each
// other).  The one barrier a tile falls between products of its last step, whose
// operands are in registers by then: behind it the next tile's stage is read
// and the stage of the tile before it is loaded.  Measured on products of 8192
// x 4096 x 16384: matrix cores 66 - 75% busy; without the loads' issue the
// kernels take 13 - 17% fewer cycles, without LDS reads as well another 5%,
// without the barrier no fewer.  (Wavefronts that load in different slots: 0 -
// 4% faster by kernel, not steadily.)
//
// Range.  A buffer resource is built per tile with the tile's own 64-bit base
// (so no operand's size is limited) and the bytes left in the operand; rows
// past the operand's end read as zeros.  A k past K inside a k-contiguous row
// is pointed out of range per lane; index-contiguous columns past the last
// read a neighbour row's values and reach only outputs that the epilogue
// drops.  Tiles past the last are loaded out of range, so that the number of
// loads in flight, which the waits count, does not depend on the tile.
#pragma once

#include "sdpa_tiles.h"
#include "xent_tiles.h"

namespace mfx {
namespace xent {

using tiles::fence;
using tiles::s16x4;
using tiles::tile_swz;

constexpr uint32_t kOOR = 0x80000000u;
constexpr int kStages = 4;

// A k-contiguous tile's rows are 64 bytes, four to the 64 banks: chunk c of row r
// at c ^ kc_swz(r) spreads the 16 rows that a 16-byte read serves at a time.
__device__ __forceinline__ int kc_swz(int r) { return (r >> 2) & 3; }

// One operand's tiles: IDX indices of a tile, NW wavefronts sharing the loads.
// KC: [IDX rows][32 k], chunk c of row r at c ^ kc_swz(r).
// else: [32 k][IDX], chunk c of row r at c ^ tile_swz<IDX>(r).
// ROT: the tiles of k are walked round from a later one (its number `at`).
template <bool KC, int IDX, int NW, bool ROT = false>
struct Tile {
  static constexpr int ELEMS = IDX * kBK16;
  static constexpr int RPI = KC ? 16 : 512 / IDX;  // rows one load instruction covers
  static constexpr int ROWS = KC ? IDX : kBK16;
  static constexpr int LOADS = ROWS / (RPI * NW);
  static_assert(LOADS >= 1 && LOADS * RPI * NW == ROWS, "whole loads");
  // Rows between instructions of a wavefront: whole swizzle periods (16), or
  // half of one, which flips bit 3 of the source chunk.
  static constexpr int STEP = RPI * NW;
  static_assert(STEP % 16 == 0 || (!KC && STEP == 8), "one or two source chunks per lane");
  static constexpr int NOFF = STEP % 16 == 0 ? 1 : 2;

  const bf16* cur;      // the next tile's first element (KC: row idx0; else: index idx0)
  int64_t next;         // elements from tile to tile
  int k0, k_end, K;     // the next tile's first k; the k to stop at
  int ld2;              // bytes from row to row
  int last;             // KC: bytes from a tile's first element to its last row's end at k 0 = 0
                        // else: bytes of the last row
  uint32_t voff[NOFF];  // this lane's byte offset in instructions 0 and 1, less the rows between
  int lane_k;           // KC: k of the lane's chunk within a tile
  int turn;             // ROT: tiles left
#if defined(__HIP_DEVICE_COMPILE__)
  __amdgpu_buffer_rsrc_t rsrc;
#endif
  uint32_t vo;          // KC: voff, or out of range past K

  // (The range check drops the whole of a load that reaches past the extent: a
  // row ends with its last chunk, whose surplus elements are zeros or meet
  // zeros; rows are whole chunks wide.)
  static __device__ __forceinline__ int chunks(int n) { return (n + 7) & ~7; }
  __device__ __forceinline__ Tile(const Operand& o, int idx0, int total, int k, int kt0, int kt1, int wave, int lane,
                                  int at = 0) {
    const int left = total - idx0;
    K = k;
    k0 = (kt0 + at) * kBK16;
    k_end = min(K, kt1 * kBK16);
    turn = kt1 - kt0;
    ld2 = (int)o.ld * 2;
    next = KC ? kBK16 : kBK16 * o.ld;
    cur = static_cast<const bf16*>(o.p) + (KC ? (int64_t)idx0 * o.ld + k0 : (int64_t)k0 * o.ld + idx0);
    last = KC ? (min(left, IDX) - 1) * ld2 + chunks(K) * 2 : chunks(left) * 2;
    constexpr int CPR = KC ? kBK16 / 8 : IDX / 8;  // chunks per row
    const int row = wave * RPI + lane / CPR, slot = lane % CPR;
    const int chunk = KC ? slot ^ kc_swz(row) : slot ^ tile_swz<IDX>(row);
    lane_k = chunk * 8;
#pragma unroll
    for (int i = 0; i < NOFF; ++i) voff[i] = (uint32_t)(row * ld2 + (chunk ^ (i * 8)) * 16);
    vo = voff[0];
  }
  // Takes up the next tile: its resource (empty past k_end), then its loads one by one.
  __device__ __forceinline__ void take() {
#if defined(__HIP_DEVICE_COMPILE__)
    int extent = KC ? last - k0 * 2 : (min(K - k0, kBK16) - 1) * ld2 + last;
    if (ROT ? turn-- <= 0 : k0 >= k_end) extent = 0;
    rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<bf16*>(cur), (short)0, extent, 0x00020000);
    if constexpr (KC) vo = k0 + lane_k < K ? voff[0] : kOOR;
    cur += next;
    k0 += kBK16;
    if constexpr (ROT) {
      static_assert(KC, "steps along a row");
      if (k0 >= k_end) {  // (one range: k from 0)
        cur -= k0;
        k0 = 0;
      }
    }
#endif
  }
  __device__ __forceinline__ void load(int i, bf16* lds, int wave) const {
#if defined(__HIP_DEVICE_COMPILE__)
    const uint32_t v = NOFF == 1 ? vo : voff[i % NOFF];
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (tiles::lds_void_t*)(lds + (NW * i + wave) * 64 * 8), 16,
                                             (NOFF == 1 && !KC ? voff[0] : v) + (uint32_t)(i * STEP * ld2), 0, 0, 0);
#endif
  }
};

// A 32 x 16 fragment: lane (l32, half) holds index l32, k = half * 8 .. + 7,
// from a k-contiguous tile one 16-byte read, from an index-contiguous one two
// transposing reads of 4 rows (k) each.
template <bool KC>
struct Frag {
  bf16x8 v;
  __device__ __forceinline__ bf16x8 bits() const { return v; }
  __device__ __forceinline__ void tie() { asm volatile("" : "+v"(v)); }
};
template <>
struct Frag<false> {
  s16x4 lo, hi;
  __device__ __forceinline__ bf16x8 bits() const {
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  __device__ __forceinline__ void tie() { asm volatile("" : "+v"(lo), "+v"(hi)); }
};

// Fragments of NB neighbouring 32-index blocks of an operand's tile.  Byte
// addresses are those of one stage; move() takes them to another.
template <bool KC, int IDX, int NB>
struct Reader {
  static constexpr int NA = KC ? 2 : 2 * NB;
  static constexpr int READS = KC ? NB : 2 * NB;  // of a step
  uint32_t a[NA];
  __device__ __forceinline__ Reader(uint32_t tile, int blk0, int lane) {
    const int half = lane >> 5, l32 = lane & 31;
    if constexpr (KC) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
        a[ks] = tile + (uint32_t)((blk0 * 32 + l32) * 64 + ((2 * ks + half) ^ kc_swz(l32)) * 16);
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
  // Read R of step KS.
  template <int KS, int R>
  __device__ __forceinline__ void read(Frag<KC> (&f)[NB]) const {
    if constexpr (KC) tiles::ds_b128<R * 2048>(f[R].v, a[KS]);
    else if constexpr (R & 1) tiles::ds_tr<KS * 16 * IDX * 2>(f[R / 2].hi, a[R]);
    else tiles::ds_tr<KS * 16 * IDX * 2>(f[R / 2].lo, a[R]);
  }
  __device__ __forceinline__ void move(uint32_t by) {
#pragma unroll
    for (int i = 0; i < NA; ++i) a[i] += by;
  }
};

// s_waitcnt vmcnt(N), other counters left alone.
template <int N>
__device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | (N >> 4) << 14);
}

// A barrier alone: __syncthreads would also wait for the loads in flight.
__device__ __forceinline__ void barrier() {
  fence();
  __builtin_amdgcn_s_barrier();
  fence();
}

// The sums of tile (m0, n0) over the k-tiles [kt0, kt1) (at least one).
template <class C>
__device__ __forceinline__ void gemm_tile16(const GemmShape& g, int m0, int n0, int kt0, int kt1, bf16* smem,
                                            Acc<C>& acc) {
  constexpr int FM = C::FM, FN = C::FN, NQ = FM * FN;  // products of a step
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % C::WM, wn = wave / C::WM;

  // Few rows against many: the reads of B set the time, and workgroups that all
  // walk the same 64 bytes of their rows crowd on a part of the memory channels
  // (rows are often a power of two apart).  Neighbouring tiles start one tile of
  // k apart: [33 x 4096] by [65537 x 4096] 151 us from the same k, 142 so; 2%
  // slower where B fits the last cache.
  constexpr bool ROT = C::ROT;
  using TA = Tile<C::A_KC, C::BM, C::NW, ROT>;
  using TB = Tile<C::B_KC, C::BN, C::NW, ROT>;
  const int at = ROT ? n0 / C::BN % (kt1 - kt0) : 0;
  constexpr int LA = TA::LOADS, NL = LA + TB::LOADS, STAGE = C::STAGE;
  TA ta(g.a, m0, g.M, g.K, kt0, kt1, wave, lane, at);
  TB tb(g.b, n0, g.N, g.K, kt0, kt1, wave, lane, at);
  const uint32_t lds = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)smem;
  using RA = Reader<C::A_KC, C::BM, FM>;
  using RB = Reader<C::B_KC, C::BN, FN>;
  RA ra(lds, wm * FM, lane);
  RB rb(lds + TA::ELEMS * 2, wn * FN, lane);
  constexpr int NR = RA::READS + RB::READS;  // reads of a step

#pragma unroll
  for (int j = 0; j < FN; ++j)
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[j][i][e] = 0.f;

  Frag<C::A_KC> fa[2][FM];
  Frag<C::B_KC> fb[2][FN];
  auto stage = [&](int kt) { return smem + ((kt - kt0) & (kStages - 1)) * (STAGE / 2); };
  // Reads and loads of product slot q: read r of step KS into set S, in order;
  // (both directions of the wait below count on their order.)
  auto read = [&](auto ks_tag, auto set_tag, auto r_tag) __attribute__((always_inline)) {
    constexpr int KS = decltype(ks_tag)::value, S = decltype(set_tag)::value, r = decltype(r_tag)::value;
    if constexpr (r < RB::READS) rb.template read<KS, r>(fb[S]);
    else ra.template read<KS, r - RB::READS>(fa[S]);
  };
  // The operands of a step have landed: their uses come after this.
  auto landed = [&](auto set_tag) __attribute__((always_inline)) {
    constexpr int S = decltype(set_tag)::value;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int j = 0; j < FN; ++j) fb[S][j].tie();
#pragma unroll
    for (int i = 0; i < FM; ++i) fa[S][i].tie();
    fence();
  };
  // The products of set S in order, with between(q) ahead of product q.
  auto multiply = [&](auto set_tag, auto between) __attribute__((always_inline)) {
    constexpr int S = decltype(set_tag)::value;
    tiles::static_for<0, NQ>([&](auto q_tag) {
      constexpr int q = decltype(q_tag)::value, j = q / FM, i = q % FM;
      between(q_tag);
      fence();
      acc[j][i] = mfma16<C::E>(fb[S][j].bits(), fa[S][i].bits(), acc[j][i]);
      fence();
    });
  };
  // Those of the reads that fall to slot q when they are spread over the slots
  // [from, to).
  auto spread = [](auto q_tag, auto from_tag, auto to_tag, auto f) __attribute__((always_inline)) {
    constexpr int q = decltype(q_tag)::value, a = decltype(from_tag)::value, b = decltype(to_tag)::value;
    if constexpr (q >= a && q < b) tiles::static_for<(q - a) * NR / (b - a), (q - a + 1) * NR / (b - a)>(f);
  };
  auto load = [&](int l, bf16* to) __attribute__((always_inline)) {
    if (l < LA) ta.load(l, to, wave);
    else tb.load(l - LA, to + TA::ELEMS, wave);
  };
  // A tile's loads go out evenly over the 2 NQ slots from one barrier to the
  // next: those of slot c.
  constexpr int B0 = NQ >= 16 ? NQ / 4 : NQ / 2;  // the slot of step 1 with the barrier
  auto slot_load = [&](auto c_tag, bf16* to) __attribute__((always_inline)) {
    constexpr int c = decltype(c_tag)::value;
#pragma unroll
    for (int l = c * NL / (2 * NQ); l < (c + 1) * NL / (2 * NQ); ++l) load(l, to);
  };
  constexpr int EARLY = (NQ - B0) * NL / (2 * NQ);  // loads of a tile that fall into step 1, behind the barrier
  // The scalar and address work goes between products too, where it is free:
  // A's next tile is taken up behind its last load, B's likewise, and the read
  // addresses move on behind step 0's reads.
  constexpr int TAKE_A = NQ * 5 / 8, MOVE_A = NQ * 3 / 4, MOVE_B = NQ * 3 / 4 + NQ / 16;
  constexpr int TAKE_B = NQ >= 4 ? NQ - 2 : NQ - 1;
  constexpr int LAST_A = (LA * 2 * NQ + NL - 1) / NL - 1;       // slot of A's last load
  constexpr int FIRST_B = ((LA + 1) * 2 * NQ + NL - 1) / NL - 1;  // and of B's first
  static_assert(LAST_A - (NQ - B0) <= TAKE_A && B0 <= TAKE_B && TAKE_B - B0 < FIRST_B && NQ / 2 <= MOVE_A,
                "behind the last use and before the next");
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using Barrier = std::integral_constant<int, B0>;
  using Half = std::integral_constant<int, NQ / 2>;
  using Most = std::integral_constant<int, B0 + NQ / 2>;

  // Three tiles, and of the fourth what falls before step 0.
  for (int t = 0; t < 3; ++t) {
    ta.take();
    tb.take();
#pragma unroll
    for (int l = 0; l < NL; ++l) load(l, stage(kt0 + t));
  }
  ta.take();
  tb.take();
#pragma unroll
  for (int l = 0; l < EARLY; ++l) load(l, stage(kt0 + 3));
  wait_loads<2 * NL + EARLY>();
  barrier();
  tiles::static_for<0, NR>([&](auto r) { read(I0{}, I0{}, r); });
  landed(I0{});
  uint32_t to = 3;  // the stage being loaded
  for (int kt = kt0; kt < kt1 - 1; ++kt) {
    bf16* const old = smem + to * (STAGE / 2);
    to = (to + 1) & (kStages - 1);
    bf16* const fresh = smem + to * (STAGE / 2);
    const uint32_t by = to == 3 ? (uint32_t)(-3 * STAGE) : (uint32_t)STAGE;
    // Step 0, reading step 1.
    multiply(I0{}, [&](auto q_tag) __attribute__((always_inline)) {
      constexpr int q = decltype(q_tag)::value;
      spread(q_tag, I0{}, Half{}, [&](auto r) { read(I1{}, I1{}, r); });
      slot_load(std::integral_constant<int, q + NQ - B0>{}, old);
      if constexpr (q == TAKE_A) ta.take();
      if constexpr (q == MOVE_A) ra.move(by);
      if constexpr (q == MOVE_B) rb.move(by);
    });
    landed(I1{});
    // Step 1.  Its operands are in registers and nobody reads this stage any
    // more; at its slot B0 tile kt + 1 has landed for everyone, and the loads
    // go on with tile kt + 4 into this one.
    multiply(I1{}, [&](auto q_tag) __attribute__((always_inline)) {
      constexpr int q = decltype(q_tag)::value;
      if constexpr (q < B0) {
        slot_load(std::integral_constant<int, q + 2 * NQ - B0>{}, old);
      } else {
        if constexpr (q == B0) {
          wait_loads<2 * NL>();
          barrier();
        }
        spread(q_tag, Barrier{}, Most{}, [&](auto r) { read(I0{}, I0{}, r); });
        slot_load(std::integral_constant<int, q - B0>{}, fresh);
        if constexpr (q == TAKE_B) tb.take();
      }
    });
    landed(I0{});
  }
  multiply(I0{}, [&](auto q_tag) __attribute__((always_inline)) {
    spread(q_tag, I0{}, Half{}, [&](auto r) { read(I1{}, I1{}, r); });
  });
  landed(I1{});
  multiply(I1{}, [](auto) {});
  wait_loads<0>();  // (those out of range: the stages are the caller's now)
}

}  // namespace xent
}  // namespace mfx

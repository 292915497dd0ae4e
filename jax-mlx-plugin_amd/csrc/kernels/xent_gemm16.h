// The 16-bit product kernel of the linear cross entropy (linear_xent.hip):
//
//   C[m][n] = sum_k A(m, k) B(n, k)        fp32 accumulation
//
// Each operand is stored either k-contiguous, [index][k], or index-contiguous,
// [k][index]; what happens to a tile's sums is the Epilogue's business (a
// softmax's partial sums, a gradient, a store).  As in gemm16.hip the kernel
// computes C^T on v_mfma_f32_32x32x16 (its A operand taken from B): an
// accumulator lane then holds one row m and 16 columns n, so a row's maximum
// and sum need one exchange between two lanes.
//
// Schedule.  Tiles of BM x BN outputs and 64 k; 256 x 256 with 8 wavefronts
// of 128 x 64 each.  Per 64 k a CU then reads 192 KB from LDS beside 2.1 us *
// its matrix rate of products, 75% of what the LDS delivers in that time
// (128 x 128 tiles with 64 x 64 a wavefront read it all and stop at 0.6-0.87
// PFLOP/s).  Two LDS stages (64 KB each at 256 x 256) are filled by LDS-DMA.  A
// k-tile is four steps of 16 k, the operands of step s + 1 read while step s
// multiplies.  The barrier sits before the last step's products, when its
// operands are in registers and the stage is free: behind it the next tile's
// first operands are read and the DMA of the tile after goes into this stage,
// both under those products.  So a k-tile's loads have a whole k-tile to
// land, and no product waits for a first LDS read.
//
// Range.  A buffer resource is built per tile with the tile's own 64-bit base
// (so no operand's size is limited) and the bytes left in the operand; rows
// past the operand's end read as zeros.  A k past K inside a k-contiguous row
// is pointed out of range per lane; index-contiguous columns past the last
// read a neighbour row's values and reach only outputs that the epilogue
// drops.
#pragma once

#include "sdpa_tiles.h"
#include "xent_tiles.h"

namespace mfx {
namespace xent {

using tiles::fence;
using tiles::s16x4;
using tiles::tile_swz;

constexpr uint32_t kOOR = 0x80000000u;

// One operand's tiles: IDX indices of a tile, NW wavefronts sharing the loads.
// KC: [IDX rows][64 k], 128 bytes a row, chunk c of row r at c ^ tile_swz<64>(r).
// else: [64 k][IDX], chunk c of row r at c ^ tile_swz<128>(r).
template <bool KC, int IDX, int NW>
struct Tile {
  static constexpr int ELEMS = IDX * kBK16;
  static constexpr int RPI = KC ? 8 : 512 / IDX;           // rows one load instruction covers
  static constexpr int ROWS = KC ? IDX : kBK16;
  static constexpr int LOADS = ROWS / (RPI * NW);
  static_assert(LOADS >= 1 && LOADS * RPI * NW == ROWS, "whole loads");
  // Rows that instructions of one wavefront are apart keep the swizzle.
  static_assert(KC ? (RPI * NW) % 8 == 0 : (RPI * NW) % 16 == 0, "one source chunk per lane");

  const bf16* base;   // KC: row idx0, k 0; else: row 0, index idx0
  int64_t ld;
  int left;           // KC: indices from idx0 on; else: the same (columns)
  int K;
  uint32_t voff;      // this lane's byte offset in instruction 0
  int lane_k;         // KC: k of the lane's chunk within a tile

  __device__ __forceinline__ Tile(const Operand& o, int idx0, int total, int k, int wave, int lane) {
    ld = o.ld;
    left = total - idx0;
    K = k;
    base = static_cast<const bf16*>(o.p) + (KC ? (int64_t)idx0 * o.ld : (int64_t)idx0);
    constexpr int CPR = KC ? 8 : IDX / 8;  // chunks per row
    const int row = wave * RPI + lane / CPR, slot = lane % CPR;
    const int chunk = KC ? slot ^ tile_swz<64>(row) : slot ^ tile_swz<128>(row);
    lane_k = chunk * 8;
    voff = (uint32_t)(((int64_t)row * ld + chunk * 8) * 2);
  }
  // (The range check drops the whole of a load that reaches past the extent: a
  // row ends with its last chunk, whose surplus elements are zeros or meet
  // zeros; rows are whole chunks wide.)
  static __device__ __forceinline__ int chunks(int n) { return (n + 7) & ~7; }
  __device__ __forceinline__ void load(int kt, bf16* lds, int wave) const {
#if defined(__HIP_DEVICE_COMPILE__)
    const int k0 = kt * kBK16;
    const bf16* from;
    int64_t extent;
    uint32_t vo = voff;
    if constexpr (KC) {
      from = base + k0;
      extent = ((int64_t)(min(left, IDX) - 1) * ld + chunks(K - k0)) * 2;
      if (k0 + lane_k >= K) vo = kOOR;
    } else {
      from = base + (int64_t)k0 * ld;
      extent = ((int64_t)(min(K - k0, kBK16) - 1) * ld + chunks(left)) * 2;
    }
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<bf16*>(from), (short)0, (int)(extent > 0x7fffffff ? 0x7fffffff : extent), 0x00020000);
    const uint32_t step = (uint32_t)(RPI * NW * ld * 2);
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (tiles::lds_void_t*)(lds + (NW * i + wave) * 64 * 8), 16,
                                               vo + (uint32_t)i * step, 0, 0, 0);
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
// addresses are those of one stage; move() takes them to the other.
template <bool KC, int IDX, int NB>
struct Reader {
  static constexpr int NA = KC ? 4 : 2 * NB;
  uint32_t a[NA];
  __device__ __forceinline__ Reader(uint32_t tile, int blk0, int lane) {
    const int half = lane >> 5, l32 = lane & 31;
    if constexpr (KC) {
      const int sw = tile_swz<64>(l32);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
        a[ks] = tile + (uint32_t)((blk0 * 32 + l32) * 128 + ((2 * ks + half) ^ sw) * 16);
    } else {
      const int tj = lane & 15, tg = (lane >> 4) & 1;
      const int r = 8 * half + (tj >> 2);
      const int chunk = tg * 2 + ((tj & 3) >> 1), sub = (tj & 1) * 8;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int c = (blk0 + b) * 4 + chunk;
        a[2 * b] = tile + (uint32_t)(r * IDX * 2 + (c ^ tile_swz<128>(r)) * 16 + sub);
        a[2 * b + 1] = tile + (uint32_t)((r + 4) * IDX * 2 + (c ^ tile_swz<128>(r + 4)) * 16 + sub);
      }
    }
  }
  template <int KS, int B>
  __device__ __forceinline__ void read(Frag<KC>& f) const {
    if constexpr (KC) {
      tiles::ds_b128<B * 4096>(f.v, a[KS]);
    } else {
      tiles::ds_tr<KS * 16 * IDX * 2>(f.lo, a[2 * B]);
      tiles::ds_tr<KS * 16 * IDX * 2>(f.hi, a[2 * B + 1]);
    }
  }
  __device__ __forceinline__ void move(uint32_t by) {
#pragma unroll
    for (int i = 0; i < NA; ++i) a[i] += by;
  }
};

// The sums of tile (m0, n0) over the k-tiles [kt0, kt1) (at least one).
template <class C>
__device__ __forceinline__ void gemm_tile16(const GemmShape& g, int m0, int n0, int kt0, int kt1, bf16* smem,
                                            Acc<C>& acc) {
  constexpr int FM = C::FM, FN = C::FN;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % C::WM, wn = wave / C::WM;

  using TA = Tile<C::A_KC, C::BM, C::NW>;
  using TB = Tile<C::B_KC, C::BN, C::NW>;
  const TA ta(g.a, m0, g.M, g.K, wave, lane);
  const TB tb(g.b, n0, g.N, g.K, wave, lane);
  bf16* const sa = smem;
  bf16* const sb = smem + TA::ELEMS;
  const uint32_t lds = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)smem;
  Reader<C::A_KC, C::BM, FM> ra(lds, wm * FM, lane);
  Reader<C::B_KC, C::BN, FN> rb(lds + TA::ELEMS * 2, wn * FN, lane);

#pragma unroll
  for (int j = 0; j < FN; ++j)
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[j][i][e] = 0.f;

  auto load = [&](int kt, int st) {
    ta.load(kt, sa + st * (C::STAGE / 2), wave);
    tb.load(kt, sb + st * (C::STAGE / 2), wave);
  };
  Frag<C::A_KC> fa[2][FM];
  Frag<C::B_KC> fb[2][FN];
  auto read = [&](auto ks_tag, int set) {
    constexpr int KS = decltype(ks_tag)::value;
    tiles::static_for<0, FN>([&](auto j) { rb.template read<KS, decltype(j)::value>(fb[set][decltype(j)::value]); });
    tiles::static_for<0, FM>([&](auto i) { ra.template read<KS, decltype(i)::value>(fa[set][decltype(i)::value]); });
  };
  // The operands of a step have landed: their uses come after this.
  auto landed = [&](int set) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int j = 0; j < FN; ++j) fb[set][j].tie();
#pragma unroll
    for (int i = 0; i < FM; ++i) fa[set][i].tie();
    fence();
  };
  auto multiply = [&](int set) {
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int i = 0; i < FM; ++i) acc[j][i] = mfma16<C::E>(fb[set][j].bits(), fa[set][i].bits(), acc[j][i]);
  };
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  using I3 = std::integral_constant<int, 3>;

  load(kt0, 0);
  tiles::wait_dma();
  __syncthreads();
  if (kt0 + 1 < kt1) load(kt0 + 1, 1);
  read(I0{}, 0);
  landed(0);
  // Steps 0 to 2; the last step's operands are in set 1 behind them.
  auto steps = [&]() __attribute__((always_inline)) {
    read(I1{}, 1);
    fence();
    multiply(0);
    landed(1);
    read(I2{}, 0);
    fence();
    multiply(1);
    landed(0);
    read(I3{}, 1);
    fence();
    multiply(0);
    landed(1);
  };
  // (The last tile runs behind the loop: with its branch inside, the sums would
  // be live in two sets of registers.)
  int by = C::STAGE;
  for (int kt = kt0; kt < kt1 - 1; ++kt) {
    steps();
    // Tile kt + 1 is in its stage, and nobody reads this one any more.
    tiles::wait_dma();
    __syncthreads();
    ra.move((uint32_t)by);
    rb.move((uint32_t)by);
    by = -by;
    read(I0{}, 0);
    if (kt + 2 < kt1) load(kt + 2, (kt - kt0) & 1);
    fence();
    multiply(1);
    landed(0);
  }
  steps();
  multiply(1);
}

}  // namespace xent
}  // namespace mfx

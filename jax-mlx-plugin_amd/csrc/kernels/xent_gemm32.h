// The f32 product kernel of the linear cross entropy: C[m][n] = sum_k A(m, k)
// B(n, k) on v_mfma_f32_32x32x2_f32, operands stored as in xent_gemm16.h, tiles
// of 32 k by 4 wavefronts: 128 x 128 outputs (64 x 64 a wavefront), 64 x 64
// where those are too few, or 32 x 32, of which each wavefront takes every
// fourth tile of k (gemm_block32).
//
// A 32x32x2 product takes 64 cycles, so the 16 (4) products per 8 k and
// wavefront leave 1024 (256) cycles for 4 to 16 (2 to 8) LDS reads: plain double
// buffering (global -> registers -> LDS, one barrier a tile), with two tiles in
// registers, keeps the matrix cores fed.
// The k of products are permuted alike in both operands: step e of 8 k takes k =
// half * 4 + e, so a k-contiguous row gives four steps in one 16-byte read.
// Rows padded by 16 bytes (k-contiguous) or 32 (index-contiguous, whose two
// halves read rows 4 apart) keep the reads off each other's banks.
#pragma once

#include <type_traits>

#include "xent_tiles.h"

namespace mfx {
namespace xent {

template <bool KC, int IDX, int NT = 256>
struct Tile32 {
  static constexpr int ROW = KC ? kBK32 + 4 : IDX + 8;        // floats
  static constexpr int CPR = KC ? kBK32 / 4 : IDX / 4;        // 16-byte chunks per row
  static constexpr int CH = IDX * kBK32 / 4 / NT;             // chunks per thread
  const float* p;
  int64_t ld;
  int idx0, total, K, tid;
  f32x4 r[2][CH];  // two tiles on their way
  __device__ __forceinline__ Tile32(const Operand& o, int i0, int n, int k)
      : p(static_cast<const float*>(o.p)), ld(o.ld), idx0(i0), total(n), K(k), tid(threadIdx.x % NT) {}
  // (K and an index-contiguous operand's rows are whole chunks, K % 4 == 0 and
  // total % 4 == 0 or the row padded to it: checked on the host.)
  __device__ __forceinline__ void load(int kt, int set) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = tid + i * NT, row = c / CPR, col = c % CPR * 4;
      const int idx = idx0 + (KC ? row : col), k = kt * kBK32 + (KC ? col : row);
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      if (idx < total && k < K) v = *reinterpret_cast<const f32x4*>(p + (KC ? idx * ld + k : k * ld + idx));
      r[set][i] = v;
    }
  }
  __device__ __forceinline__ void store(float* lds, int set) const {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = tid + i * NT, row = c / CPR, col = c % CPR * 4;
      *reinterpret_cast<f32x4*>(lds + row * ROW + col) = r[set][i];
    }
  }
};

// The four k of step c (of 8) that this lane's half holds, for index `idx`.
template <bool KC, int IDX, int NT = 256>
__device__ __forceinline__ f32x4 frag32(const float* lds, int idx, int c, int half) {
  constexpr int ROW = Tile32<KC, IDX, NT>::ROW;
  const int k = c * 8 + half * 4;
  if constexpr (KC) return *reinterpret_cast<const f32x4*>(lds + idx * ROW + k);
  else return f32x4{lds[k * ROW + idx], lds[(k + 1) * ROW + idx], lds[(k + 2) * ROW + idx], lds[(k + 3) * ROW + idx]};
}

template <class C>
__device__ __forceinline__ void gemm_tile32(const GemmShape& g, int m0, int n0, int kt0, int kt1, float* smem,
                                            Acc<C>& acc) {
  static_assert(C::BM == C::BN && C::NT == 256, "square tiles by four wavefronts");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, l32 = lane & 31;
  const int wm = wave % C::WM, wn = wave / C::WM;
  Tile32<C::A_KC, C::BM> ta(g.a, m0, g.M, g.K);
  Tile32<C::B_KC, C::BN> tb(g.b, n0, g.N, g.K);
  constexpr int HALF = C::STAGE / 8;  // floats of one operand's tile
#pragma unroll
  for (int j = 0; j < C::FN; ++j)
#pragma unroll
    for (int i = 0; i < C::FM; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[j][i][e] = 0.f;
  // Tile kt multiplies from its LDS stage while kt + 1 is in registers (stored
  // at the end) and kt + 2 on its way: a tile's products alone (1024 cycles at
  // 64 x 64) do not cover a load.
  ta.load(kt0, 0);
  tb.load(kt0, 0);
  ta.load(kt0 + 1, 1);  // (past K: zeros)
  tb.load(kt0 + 1, 1);
  ta.store(smem, 0);
  tb.store(smem + HALF, 0);
  __syncthreads();
  auto tile = [&](int kt, auto set_tag) __attribute__((always_inline)) {
    constexpr int S = decltype(set_tag)::value;  // kt's stage and, for kt + 2, register set
    const float* at = smem + S * 2 * HALF;
    const float* bt = at + HALF;
    float* const next = smem + (S ^ 1) * 2 * HALF;
    ta.load(kt + 2, S);
    tb.load(kt + 2, S);
#pragma unroll
    for (int c = 0; c < kBK32 / 8; ++c) {
      f32x4 fa[C::FM], fb[C::FN];
#pragma unroll
      for (int i = 0; i < C::FM; ++i) fa[i] = frag32<C::A_KC, C::BM>(at, (wm * C::FM + i) * 32 + l32, c, half);
#pragma unroll
      for (int j = 0; j < C::FN; ++j) fb[j] = frag32<C::B_KC, C::BN>(bt, (wn * C::FN + j) * 32 + l32, c, half);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int j = 0; j < C::FN; ++j)
#pragma unroll
          for (int i = 0; i < C::FM; ++i)
            acc[j][i] = __builtin_amdgcn_mfma_f32_32x32x2f32(fb[j][e], fa[i][e], acc[j][i], 0, 0, 0);
    }
    ta.store(next, S ^ 1);
    tb.store(next + HALF, S ^ 1);
    __syncthreads();
  };
  int kt = kt0;
  for (; kt + 1 < kt1; kt += 2) {
    tile(kt, std::integral_constant<int, 0>{});
    tile(kt + 1, std::integral_constant<int, 1>{});
  }
  if (kt < kt1) tile(kt, std::integral_constant<int, 0>{});
}

// A block of 32 x 32 outputs whose tiles of k the wavefronts take in turn, for
// products too small to fill the CUs otherwise: a 64 x 64 tile keeps a CU's
// matrix cores busy for 1024 cycles per 32 k, this one for 256.  Each wavefront
// turns its tiles round in an LDS stage of its own, without barriers.
// Measured, forward of [T, H] by [V, H], blocks against 64 x 64 (us): 257, 512,
// 1000: 18.6 and 22.9; 33, 1024, 8000: 26.5 and 35.3; 100, 2048, 300: 25 and 54;
// but 1000, 1024, 8000: 198 and 161 (147 in 128 x 128).  Operands straight from
// memory to the registers they multiply from were slower than through LDS (the
// last: 312; rows are read 32 bytes at a time then).
template <class C>
__device__ __forceinline__ void gemm_block32(const GemmShape& g, int m0, int n0, int kt0, int kt1, float* smem,
                                             Acc<C>& acc) {
  static_assert(C::BM == 32 && C::BN == 32 && C::KW == 4, "one block by four wavefronts");
  const int lane = threadIdx.x & 63, half = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  f32x16& a = acc[0][0];
#pragma unroll
  for (int e = 0; e < 16; ++e) a[e] = 0.f;
  constexpr int HALF = C::STAGE / 8;  // floats of one operand's tile
  float* const at = smem + wave * 2 * HALF;
  float* const bt = at + HALF;
  Tile32<C::A_KC, 32, 64> ta(g.a, m0, g.M, g.K);
  Tile32<C::B_KC, 32, 64> tb(g.b, n0, g.N, g.K);
  // (One wavefront: its LDS operations are in order.)
  auto in_order = [] {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  auto tile = [&](int kt, int set) __attribute__((always_inline)) {
    ta.store(at, set);
    tb.store(bt, set);
    in_order();
    ta.load(kt + 8, set);
    tb.load(kt + 8, set);
#pragma unroll
    for (int c = 0; c < kBK32 / 8; ++c) {
      const f32x4 fa = frag32<C::A_KC, 32, 64>(at, l32, c, half), fb = frag32<C::B_KC, 32, 64>(bt, l32, c, half);
#pragma unroll
      for (int e = 0; e < 4; ++e) a = __builtin_amdgcn_mfma_f32_32x32x2f32(fb[e], fa[e], a, 0, 0, 0);
    }
    in_order();
  };
  int kt = kt0 + wave;
  ta.load(kt, 0);  // (past K: zeros)
  tb.load(kt, 0);
  ta.load(kt + 4, 1);
  tb.load(kt + 4, 1);
  for (; kt < kt1; kt += 8) {
    tile(kt, 0);
    if (kt + 4 < kt1) tile(kt + 4, 1);
  }
  // The others' sums, added in order.
  __syncthreads();
  f32x4* const sums = reinterpret_cast<f32x4*>(smem);
  if (wave > 0)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      sums[((wave - 1) * 4 + q) * 64 + lane] = f32x4{a[q * 4], a[q * 4 + 1], a[q * 4 + 2], a[q * 4 + 3]};
  __syncthreads();
  if (wave == 0)
#pragma unroll
    for (int w = 0; w < 3; ++w)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 v = sums[(w * 4 + q) * 64 + lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) a[q * 4 + e] += v[e];
      }
}

}  // namespace xent
}  // namespace mfx

// Shapes shared by the product kernels of the linear cross entropy
// (xent_gemm16.h, xent_gemm32.h) and their epilogues (linear_xent.hip).
#pragma once

#include "sdpa_elem.h"

namespace mfx {
namespace xent {

constexpr int kBK16 = 32, kBK32 = 32;  // k per tile

struct Operand {
  const void* p;
  int64_t ld;  // elements from one row (k-contiguous: index; else k) to the next
};

struct GemmShape {
  Operand a, b;
  int M, N, K;
  int tiles_m, tiles_n;
  int splits;        // k-ranges per output tile (grid = tiles * splits)
  int kt_per_split;  // k-tiles per range
};

// (tile row, tile column) of a workgroup.  Workgroups are dealt to the 8 XCDs
// in turn: each XCD takes a run of tiles of its own, walked in bands of 8
// tile rows, so that the 32 tiles it works on at a time share 8 + 4 operand
// panels in its L2.
__device__ __forceinline__ void map_tile(int id, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int n = tiles_m * tiles_n;
  const int per = n >> 3, rest = n & 7, xcd = id & 7;
  int t = (id >> 3) + xcd * per + min(xcd, rest);
  const int band = 8 * tiles_n;
  const int b = t / band;
  const int rows = min(8, tiles_m - b * 8);
  t -= b * band;
  tm = b * 8 + t % rows;
  tn = t / rows;
}

// E: 0 bf16, 1 f16, 2 f32.  KW wavefronts share each block's k; the first of
// them (wave < WM * WN) ends with the sums.
template <int BM_, int BN_, int WM_, int WN_, bool A_KC_, bool B_KC_, int E_, int KW_ = 1>
struct Config {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, E = E_, KW = KW_;
  static constexpr bool A_KC = A_KC_, B_KC = B_KC_;
  static constexpr int NW = WM * WN * KW, NT = NW * 64;
  static constexpr int WAVES = BM == 256 ? 1 : BM == 128 ? 2 : BM == 64 ? 3 : 4;  // per SIMD
  static constexpr int FM = BM / (32 * WM), FN = BN / (32 * WN);  // blocks of a wavefront
  static constexpr int BK = E == 2 ? kBK32 : kBK16;
  // Bytes of a stage, and of all: four in 16 bits; f32: two, in the larger of
  // the two forms' padded rows (xent_gemm32.h).
  static constexpr int STAGE = E == 2 ? 2 * BM * (kBK32 + (BM < 128 ? 8 : 4)) * 4 : (BM + BN) * kBK16 * 2;
  // With KW > 1 one for each wavefront.
  static constexpr int SMEM = (KW > 1 ? KW : E == 2 ? 2 : 4) * STAGE;
};

template <class C>
using Acc = f32x16[C::FN][C::FM];

}  // namespace xent
}  // namespace mfx

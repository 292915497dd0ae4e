// Softmax cross entropy of a linear head, logits z = h W^T never stored:
//
//   lse_t = log sum_v exp(z_tv),  loss_t = lse_t - z_t,target(t)
//   d_tv  = (exp(z_tv - lse_t) - [v = target(t)]) * dloss_t
//   dh = d W,  dW = d^T h
//
// h [T, H] and W [V, H] in bf16, f16 or f32; all sums and the softmax in fp32.
//
// Forward: the product kernel (xent_gemm16.h, xent_gemm32.h) over tiles of
// T x V whose epilogue leaves each row's maximum and sum of exponentials over
// the tile's columns, and the target's logit; xent_combine folds a row's tiles.
// The partials are 8 bytes per row and tile of 32 to 256 columns.
//
// Backward, in pieces of the vocabulary: the piece's logits again, whose
// epilogue turns them into d, rounded to the inputs' type, in a workspace of
// T x piece (f32 for f32 inputs, nothing is rounded there); then dW of the
// piece = d^T h and dh (+)= d W of the piece.  A piece is as wide as kPieceBytes
// of d allow, so that the fp32 dh is added to in few rounds and its products
// are long.  Rounding d costs half a step of
// each entry (independent from entry to entry), as rounding the gradient of
// stored 16-bit logits would; the target's entry is rounded after the
// subtraction.  d is held over the largest |dloss|, c, which the sums are
// multiplied by at the end: with the usual equal weights the target's entry is
// p - 1 then, which for an unlikely target rounds to -1 almost exactly, where
// (p - 1) dloss would carry dloss's own rounding into every row alike
// (8192 x 4096 x 65537: dh and dW off by 0.0028 of their size with it, 0.0019
// without, 0.0017 of which is their own rounding; an f32 dW by 0.0010).  Two
// terms of d would take that away for twice the products of dh and dW.  f16
// holds d times 2^15 besides, or entries below 2^-24 would be lost.
//
// What bounds it: the matrix cores, 2 T H V flops a product, one product
// forward and three backward.  bf16, T 8192, H 4096, V 65537: forward 3.6 ms (1.22
// PFLOP/s, matrix cores 71% busy), backward 11.0 ms (1.20; logits 63%, dW 66%, dh
// 73%); a library product of these sizes runs at 1.25 - 1.58 beside them, by the
// clock.  T 4096, H 2048, V 32000: 0.47 and 1.41 ms (1.13, 1.14).  Few rows
// (T 33) read W once: 131 us for 537 MB, 4.1 TB/s.
#include <algorithm>
#include <cmath>
#include <string>

#include "xent_gemm16.h"
#include "xent_gemm32.h"

namespace mfx {
namespace xent {

// Tile forms: 256 x 256, one workgroup a CU; 128 x 128, two; 64 rows of A by
// 128 of B (f32: 64 x 64), three; and 32 x 32, four.  16 bits have the first
// three, f32 the last three.
enum Form { kWide, kNarrow, kSlim, kBlock };
constexpr int kFormM[4] = {256, 128, 64, 32};
constexpr int kFormN[2][4] = {{256, 128, 128, 0}, {0, 128, 64, 32}};  // 16 bits, f32

template <Form F, bool A_KC, bool B_KC, int E>
struct Pick;
template <bool A_KC, bool B_KC, int E>
struct Pick<kWide, A_KC, B_KC, E> : Config<256, 256, 2, 2, A_KC, B_KC, E> {};
template <bool A_KC, bool B_KC, int E>
struct Pick<kNarrow, A_KC, B_KC, E> : Config<128, 128, 2, 2, A_KC, B_KC, E> {};
template <bool A_KC, bool B_KC, int E>
struct Pick<kSlim, A_KC, B_KC, E> : Config<64, 128, 1, 4, A_KC, B_KC, E> {};
template <bool A_KC, bool B_KC>
struct Pick<kSlim, A_KC, B_KC, 2> : Config<64, 64, 2, 2, A_KC, B_KC, 2> {};
template <bool A_KC, bool B_KC>
struct Pick<kBlock, A_KC, B_KC, 2> : Config<32, 32, 1, 1, A_KC, B_KC, 2, 4> {};

template <class C>
__device__ __forceinline__ void gemm_tile(const GemmShape& g, int m0, int n0, int kt0, int kt1, char* smem,
                                          Acc<C>& acc) {
  if constexpr (C::KW > 1) gemm_block32<C>(g, m0, n0, kt0, kt1, reinterpret_cast<float*>(smem), acc);
  else if constexpr (C::E == 2) gemm_tile32<C>(g, m0, n0, kt0, kt1, reinterpret_cast<float*>(smem), acc);
  else gemm_tile16<C>(g, m0, n0, kt0, kt1, reinterpret_cast<bf16*>(smem), acc);
}

struct LossArgs {
  GemmShape g;
  const void* targets;
  int target64;
  int64_t v0;            // the piece's first column (backward)
  int V;                 // columns in all
  // forward
  float* part_m;         // [tiles_n][T], log2 units
  float* part_l;
  float* picked;         // [T]: the target's logit
  // backward
  const float* lse;
  const float* weight;   // dloss, in 16 bits over c (times 2^15)
  void* d;               // [T][ldd]
  int64_t ldd;
};

struct StoreArgs {
  GemmShape g;
  float* part;           // fp32 sums [splits][M][N], or null: store to c
  int add;               // part += instead of part =
  void* c;               // [M][ldc]
  int64_t ldc;
  int c_f32;             // c is fp32, else the inputs' type
  const float* scale;    // multiplies c (null: 1)
};

__device__ __forceinline__ int64_t target_of(const void* t, int wide, int row) {
  return wide ? static_cast<const int64_t*>(t)[row] : static_cast<const int32_t*>(t)[row];
}

// Column, within a wavefront's, of accumulator element e of block j.
__device__ __forceinline__ int column(int j, int e, int half) { return j * 32 + (e >> 2) * 8 + half * 4 + (e & 3); }

// ---- the logits' tiles -------------------------------------------------------

template <class C, bool BWD>
__global__ __launch_bounds__(C::NT, C::WAVES) void xent_logits_kernel(LossArgs p) {
  constexpr int FM = C::FM, FN = C::FN;
  __shared__ __attribute__((aligned(16))) char smem[C::SMEM];
  int tm, tn;
  map_tile(blockIdx.x, p.g.tiles_m, p.g.tiles_n, tm, tn);
  const int m0 = tm * C::BM, n0 = tn * C::BN;
  Acc<C> acc;
  gemm_tile<C>(p.g, m0, n0, 0, (p.g.K + C::BK - 1) / C::BK, smem, acc);
  __syncthreads();  // the stages are free

  const int lane = threadIdx.x & 63, half = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % C::WM, wn = wave / C::WM % C::WN;
  // (Wavefronts without sums have no rows.)
  const int M = wave < C::WM * C::WN ? p.g.M : 0, N = p.g.N;
  const int nw = n0 + wn * FN * 32;  // this wavefront's first column (of the piece)
  // Block i's values, -inf in columns past N (of which only the last tile has
  // any): 16 FN registers at a time, and the fences between blocks keep it so.
  auto block = [&](int i, auto edge_tag, float (&z)[FN * 16]) __attribute__((always_inline)) {
    fence();
    int left = N - nw - half * 4;  // (opaque, so that no comparison is kept from block to block)
    asm volatile("" : "+v"(left));
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        z[j * 16 + e] = acc[j][i][e];
        if (decltype(edge_tag)::value && column(j, e, 0) >= left) z[j * 16 + e] = -INFINITY;
      }
  };
  // The logit of this lane's column `t` (one of two lanes has it): few rows
  // have their target in a wavefront's columns, so the others need not look.
  auto pick = [&](const float (&z)[FN * 16], int64_t t, bool& mine) __attribute__((always_inline)) {
    const int n = (int)(t - nw) - half * 4;
    float x = 0.f;
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) x = column(j, e, 0) == n ? z[j * 16 + e] : x;
    mine = n >= 0 && n < FN * 32 && (n & 4) == 0;
    return x;
  };
  auto here = [&](int64_t t) { return __ballot(t >= nw && t < nw + FN * 32) != 0; };

  if constexpr (!BWD) {
    float* const red_m = reinterpret_cast<float*>(smem);  // [WN][BM]
    float* const red_l = red_m + C::WN * C::BM;
    auto fold = [&](auto edge_tag) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int r = wm * FM * 32 + i * 32 + l32, row = m0 + r;
        const int64_t t = row < M ? target_of(p.targets, p.target64, row) : -1;
        float z[FN * 16];
        block(i, edge_tag, z);
        if (here(t)) {
          bool mine;
          const float x = pick(z, t, mine);
          if (mine) p.picked[row] = x;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int e = 0; e < FN * 16; ++e) mx = fmaxf(mx, z[e]);
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float base = mx == -INFINITY ? 0.f : mx * kLog2e;
        float l[2] = {0.f, 0.f};
#pragma unroll
        for (int e = 0; e < FN * 16; ++e) l[e & 1] += __builtin_amdgcn_exp2f(fmaf(z[e], kLog2e, -base));
        l[0] += l[1];
        l[0] += __shfl_xor(l[0], 32, 64);
        if (half == 0 && (C::KW == 1 || row < M)) {
          red_m[wn * C::BM + r] = mx == -INFINITY ? mx : base;
          red_l[wn * C::BM + r] = l[0];
        }
      }
    };
    if (n0 + C::BN > N) fold(std::true_type{});
    else fold(std::false_type{});
    __syncthreads();
    for (int r = threadIdx.x; r < C::BM; r += C::NT) {
      if (m0 + r >= M) continue;
      float mx = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < C::WN; ++w) mx = fmaxf(mx, red_m[w * C::BM + r]);
      const float base = mx == -INFINITY ? 0.f : mx;
#pragma unroll
      for (int w = 0; w < C::WN; ++w) l += red_l[w * C::BM + r] * __builtin_amdgcn_exp2f(red_m[w * C::BM + r] - base);
      p.part_m[(int64_t)tn * M + m0 + r] = mx;
      p.part_l[(int64_t)tn * M + m0 + r] = l;
    }
  } else {
    // 16 bits: through LDS, whole rows of the wavefront's block at a time: 16-byte
    // chunk c of row r at slot c ^ (r % chunks).  d's rows are whole tiles
    // wide, so only rows need a check.
    constexpr int CPR = FN * 4;    // chunks per row
    constexpr int RPS = 64 / CPR;  // rows per store instruction
    bf16* const st = reinterpret_cast<bf16*>(smem) + wave * (FM * 32) * (FN * 32);
    auto turn = [&](auto edge_tag) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        int l = l32;  // (opaque: no address of a later block is formed early)
        asm volatile("" : "+v"(l));
        const int r = i * 32 + l, row = m0 + wm * FM * 32 + r;
        int64_t t = row < M ? target_of(p.targets, p.target64, row) : -1;
        const bool counts = t >= 0 && t < p.V;
        t = counts ? t - p.v0 : -1;
        const float lse2 = row < M ? p.lse[row] * kLog2e : 0.f;
        const float w = counts ? p.weight[row] : 0.f;
        auto prob = [&](float x) __attribute__((always_inline)) { return __builtin_amdgcn_exp2f(fmaf(x, kLog2e, -lse2)); };
        float z[FN * 16];
        block(i, edge_tag, z);
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            float o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = counts ? prob(z[j * 16 + g * 4 + e]) * w : 0.f;
            if constexpr (C::E == 2) {
              if (row < M)
                *reinterpret_cast<f32x4*>(static_cast<float*>(p.d) + (int64_t)row * p.ldd + nw +
                                          column(j, g * 4, half)) = f32x4{o[0], o[1], o[2], o[3]};
            } else {
              const int c = j * 4 + g;
              *reinterpret_cast<u32x2*>(st + r * (FN * 32) + (c ^ (r & (CPR - 1))) * 8 + half * 4) =
                  u32x2{pack2<C::E & 1>(o[0], o[1]), pack2<C::E & 1>(o[2], o[3])};
            }
          }
        // The target's entry, over the one just written.
        if (here(t)) {
          bool mine;
          const float d = (prob(pick(z, t, mine)) - 1.f) * w;
          const int n = (int)t - nw;
          if (mine) {
            if constexpr (C::E == 2) static_cast<float*>(p.d)[(int64_t)row * p.ldd + t] = d;
            else
              reinterpret_cast<uint16_t*>(st)[r * (FN * 32) + ((n >> 3) ^ (r & (CPR - 1))) * 8 + (n & 7)] =
                  store_e<C::E & 1>(d);
          }
        }
      }
    };
    if (n0 + C::BN > N) turn(std::true_type{});
    else turn(std::false_type{});
    if constexpr (C::E == 2) return;
    const int mw = m0 + wm * FM * 32;
#pragma unroll
    for (int k = 0; k < FM * 32 / RPS; ++k) {
      const int r = k * RPS + lane / CPR, c = lane % CPR;
      const u32x4 v = *reinterpret_cast<const u32x4*>(st + r * (FN * 32) + (c ^ (r & (CPR - 1))) * 8);
      if (mw + r < M)
        *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p.d) + (int64_t)(mw + r) * p.ldd + nw + c * 8) = v;
    }
  }
}

// lse and loss of each row from its tiles' partials: 64 rows a workgroup, a
// row's tiles shared out over 16 wavefronts, four of them in flight at a time.
constexpr int kCombine = 16;
__global__ __launch_bounds__(64 * kCombine) void xent_combine(const float* __restrict__ part_m,
                                                              const float* __restrict__ part_l,
                                                              const float* __restrict__ picked, const void* targets,
                                                              int target64, int T, int V, int tiles, float* loss,
                                                              float* lse) {
  __shared__ float red_m[kCombine][64], red_l[kCombine][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int row = blockIdx.x * 64 + lane;
  float m = -INFINITY, l = 0.f;
  if (row < T)
    for (int i0 = w; i0 < tiles; i0 += 4 * kCombine) {
      float mi[4], li[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * kCombine;
        mi[u] = i < tiles ? part_m[(int64_t)i * T + row] : -INFINITY;
        li[u] = i < tiles ? part_l[(int64_t)i * T + row] : 0.f;
      }
      // (A NaN maximum is lost to fmaxf; its sum is NaN and stays.)
      const float mn = fmaxf(fmaxf(fmaxf(mi[0], mi[1]), fmaxf(mi[2], mi[3])), m), base = mn == -INFINITY ? 0.f : mn;
      l *= __builtin_amdgcn_exp2f(m - base);
#pragma unroll
      for (int u = 0; u < 4; ++u) l += li[u] * __builtin_amdgcn_exp2f(mi[u] - base);
      m = mn;
    }
  red_m[w][lane] = m;
  red_l[w][lane] = l;
  __syncthreads();
  if (w != 0 || row >= T) return;
#pragma unroll
  for (int i = 1; i < kCombine; ++i) m = fmaxf(m, red_m[i][lane]);
  const float base = m == -INFINITY ? 0.f : m;
  l = 0.f;
#pragma unroll
  for (int i = 0; i < kCombine; ++i) l += red_l[i][lane] * __builtin_amdgcn_exp2f(red_m[i][lane] - base);
  // log(sum exp z) = m ln 2 + log(sum of 2^(z - m)).
  const float z = fmaf(m, 0.6931471805599453f, __logf(l));
  if (lse) lse[row] = z;
  const int64_t t = target_of(targets, target64, row);
  loss[row] = t >= 0 && t < V ? z - picked[row] : 0.f;
}

// weight[t] = dloss[t] / c * times for the rows that count, c their largest
// |dloss| (1 if that is 0 or not finite); *scale = c / times.
__global__ __launch_bounds__(1024) void xent_weights(const float* __restrict__ dloss, const void* targets,
                                                     int target64, int T, int V, float times, float* weight,
                                                     float* scale) {
  __shared__ float red[16];
  float m = 0.f;
  // (Eight rows in flight at a time.)
  for (int i0 = threadIdx.x; i0 < T; i0 += 8 * 1024) {
    float g[8];
    int64_t t[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = min(i0 + u * 1024, T - 1);
      g[u] = dloss[i];
      t[u] = target_of(targets, target64, i);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (t[u] >= 0 && t[u] < V) m = fmaxf(m, fabsf(g[u]));
  }
  m = group_max<64>(m);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  m = red[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) m = fmaxf(m, red[i]);
  const float c = m > 0.f && m < INFINITY ? m : 1.f;
  for (int i0 = threadIdx.x; i0 < T; i0 += 8 * 1024) {
    float g[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) g[u] = dloss[min(i0 + u * 1024, T - 1)];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i0 + u * 1024 < T) weight[i0 + u * 1024] = g[u] / c * times;
  }
  if (threadIdx.x == 0) *scale = c / times;
}

// ---- the gradients' products -------------------------------------------------

template <class C>
__global__ __launch_bounds__(C::NT, C::WAVES) void xent_grad_kernel(StoreArgs p) {
  constexpr int FM = C::FM, FN = C::FN;
  __shared__ __attribute__((aligned(16))) char smem[C::SMEM];
  const int ntiles = p.g.tiles_m * p.g.tiles_n;
  const int sp = blockIdx.x / ntiles;
  int tm, tn;
  map_tile(blockIdx.x % ntiles, p.g.tiles_m, p.g.tiles_n, tm, tn);
  const int m0 = tm * C::BM, n0 = tn * C::BN;
  const int kt0 = sp * p.g.kt_per_split;
  const int kt1 = min((p.g.K + C::BK - 1) / C::BK, kt0 + p.g.kt_per_split);
  Acc<C> acc;
  gemm_tile<C>(p.g, m0, n0, kt0, kt1, smem, acc);

  const int lane = threadIdx.x & 63, half = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % C::WM, wn = wave / C::WM % C::WN;
  // (Wavefronts without sums have no rows.)
  const int M = wave < C::WM * C::WN ? p.g.M : 0, N = p.g.N;
  const int mw = m0 + wm * FM * 32, nw = n0 + wn * FN * 32;
  const float mul = p.scale ? *p.scale : 1.f;
  if (C::E == 2 || p.part || p.c_f32) {
    float* const out = p.part ? p.part + (int64_t)sp * M * N : static_cast<float*>(p.c);
    const int64_t ld = p.part ? N : p.ldc;
    const float f = p.part ? 1.f : mul;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int m = mw + i * 32 + l32;
      if (m >= M) continue;
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int n = nw + j * 32 + g * 8 + half * 4;
          if (n >= N) continue;  // (N % 4 == 0)
          f32x4* const at = reinterpret_cast<f32x4*>(out + (int64_t)m * ld + n);
          f32x4 v = {acc[j][i][g * 4] * f, acc[j][i][g * 4 + 1] * f, acc[j][i][g * 4 + 2] * f,
                     acc[j][i][g * 4 + 3] * f};
          if (p.part && p.add) v += *at;
          *at = v;
        }
    }
    return;
  }
  if constexpr (C::E != 2) {
  __syncthreads();  // the stages are free
  constexpr int CPR = FN * 4, RPS = 64 / CPR;
  bf16* const st = reinterpret_cast<bf16*>(smem) + wave * (FM * 32) * (FN * 32);
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int r = i * 32 + l32;
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        u16x4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = store_e<C::E>(acc[j][i][g * 4 + e] * mul);
        const int c = j * 4 + g;
        *reinterpret_cast<u16x4*>(st + r * (FN * 32) + (c ^ (r & (CPR - 1))) * 8 + half * 4) = o;
      }
  }
#pragma unroll
  for (int k = 0; k < FM * 32 / RPS; ++k) {
    const int r = k * RPS + lane / CPR, c = lane % CPR;
    const u32x4 v = *reinterpret_cast<const u32x4*>(st + r * (FN * 32) + (c ^ (r & (CPR - 1))) * 8);
    if (mw + r < M && nw + c * 8 < N)
      __builtin_nontemporal_store(
          v, reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p.c) + (int64_t)(mw + r) * p.ldc + nw + c * 8));
  }
  }
}

// c = the fp32 sums of the ranges, added in order, times c.
template <typename T>
__global__ __launch_bounds__(256) void xent_sum(const float* __restrict__ part, int splits, int64_t M, int N, T* c,
                                                int64_t ldc, const float* scale) {
  for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < M * N / 4; q += (int64_t)gridDim.x * 256) {
    const int64_t e = q * 4, m = e / N, n = e % N;
    f32x4 v = *reinterpret_cast<const f32x4*>(part + e);
    for (int s = 1; s < splits; ++s) v += *reinterpret_cast<const f32x4*>(part + s * M * N + e);
    const float mul = scale ? *scale : 1.f;
    typedef T t4 __attribute__((ext_vector_type(4)));
    t4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = from_f32<T>(v[j] * mul);
    *reinterpret_cast<t4*>(c + m * ldc + n) = o;
  }
}

// ---- host ----------------------------------------------------------------------

namespace {

constexpr size_t kPieceBytes = 512u << 20;      // of d at a time
constexpr int64_t kMaxStride = int64_t(1) << 21;  // a tile's 256 rows are addressed within 31 bits

size_t align256(size_t n) { return (n + 255) / 256 * 256; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Workgroups of 256 for `n` threads' work; the kernel's threads go on in
// strides of the grid past 2^28 (a launch holds fewer than 2^32).
dim3 strided_grid(int64_t n) { return dim3((unsigned)std::min<int64_t>(ceil_div(n, 256), 1 << 20)); }

// A product's tile form and, for a gradient's, its ranges of k.
struct Way {
  Form form;
  int64_t range, ranges;  // k-tiles of one, and their number
};

// A type's first and last form.
constexpr int first_form(int E) { return E == 2 ? kNarrow : kWide; }
constexpr int last_form(int E) { return E == 2 ? kBlock : kSlim; }

GemmShape shape(Operand a, Operand b, int64_t M, int64_t N, int64_t K, int E, Form f) {
  GemmShape g{};
  g.a = a;
  g.b = b;
  g.M = (int)M;
  g.N = (int)N;
  g.K = (int)K;
  g.tiles_m = (int)ceil_div(M, kFormM[f]);
  g.tiles_n = (int)ceil_div(N, kFormN[E == 2][f]);
  g.splits = 1;
  return g;
}

// Microseconds that a form takes: a k-tile with `slots` workgroups on each CU,
// each further round of workgroups, and once.  Fitted to the measured times of
// 18 shapes from [33 x 4096 x 65537] to [8192 x 512 x 1000] in every form and
// with 1 to 16 ranges; the chosen way took at most 13% more than the best of
// them.
struct Cost {
  int slots;
  float kt, each, once;
};
constexpr Cost kCost[2][4] = {{{1, 0.85f, 9.f, 0.f}, {2, 0.57f, 1.f, 6.f}, {3, 0.85f, 0.5f, 4.f}, {}},
                              {{}, {2, 4.6f, 2.f, 6.f}, {3, 1.95f, 1.f, 4.f}, {4, 0.8f, 1.f, 4.f}}};

float way_us(const Cost& c, int64_t wgs, int64_t range, int64_t cus) {
  const int64_t full = wgs / (c.slots * cus), rest = wgs % (c.slots * cus);
  float t = c.once + (float)full * ((float)range * c.kt + c.each);
  // (With fewer than `slots` workgroups on a CU each runs faster.)
  if (rest) t += (float)range * c.kt * (0.25f + 0.75f * (float)ceil_div(rest, cus) / (float)c.slots) + c.each;
  return t;
}

// The way that takes least by these: every form, and with `split` every number
// of ranges up to 32 of at least 8 k-tiles, whose sums are written and read
// again (8 bytes an output and range at 4 TB/s, and a launch more).
Way choose(int E, int64_t M, int64_t N, int64_t K, bool split) {
  const int64_t kt = ceil_div(K, E == 2 ? kBK32 : kBK16), cus = device_cu_count();
  Way best{kNarrow, kt, 1};
  float least = INFINITY;
  for (int f = first_form(E); f <= last_form(E); ++f) {
    const Cost& c = kCost[E == 2][f];
    const int64_t tiles = ceil_div(M, kFormM[f]) * ceil_div(N, kFormN[E == 2][f]);
    for (int64_t s = 1; s <= (split ? std::min<int64_t>(32, std::max<int64_t>(1, kt / 8)) : 1); ++s) {
      const int64_t range = ceil_div(kt, s), ranges = ceil_div(kt, range);
      if (!launch_fits(tiles * ranges, 256)) continue;
      float t = way_us(c, tiles * ranges, range, cus);
      if (ranges > 1) t += 4.f + (float)ranges * (float)M * (float)N * 8.f / 4e6f;
      if (t < least) {
        least = t;
        best = Way{(Form)f, range, ranges};
      }
    }
  }
  return best;
}

struct BwdPlan {
  int E;
  int64_t piece, pieces;
  Way dh, dw;  // of the first piece, the widest
  size_t row_bytes, d_bytes, dh_bytes, dw_bytes, total;
};

int elem_of(int dtype) { return dtype == MFX_F32 ? 2 : dtype == MFX_F16 ? 1 : 0; }

BwdPlan plan_bwd(const mfx_linear_xent_bwd_args& a) {
  BwdPlan pl{};
  pl.E = elem_of(a.dtype);
  const int size = dtype_size(a.dtype);
  const int64_t vp = ceil_div(a.V, 256) * 256;
  int64_t most = std::max<int64_t>(256, (int64_t)(kPieceBytes / size) / a.T / 256 * 256);
  most = std::min(most, kMaxStride);
  pl.pieces = ceil_div(vp, most);
  pl.piece = ceil_div(ceil_div(vp, pl.pieces), 256) * 256;
  pl.pieces = ceil_div(vp, pl.piece);
  const int64_t nv = std::min(pl.piece, a.V);
  pl.d_bytes = align256((size_t)a.T * pl.piece * size);
  if (a.dh) {
    pl.dh = choose(pl.E, a.T, a.H, nv, true);
    if (pl.pieces > 1 || pl.dh.ranges > 1) pl.dh_bytes = align256((size_t)pl.dh.ranges * a.T * a.H * 4);
  }
  if (a.dw) {
    pl.dw = choose(pl.E, nv, a.H, a.T, true);
    if (pl.dw.ranges > 1) pl.dw_bytes = align256((size_t)pl.dw.ranges * nv * a.H * 4);
  }
  if (pl.E != 2) pl.row_bytes = 256 + align256((size_t)a.T * 4);
  pl.total = pl.row_bytes + pl.d_bytes + pl.dh_bytes + pl.dw_bytes;
  return pl;
}

template <int E, bool BWD>
int launch_logits(const LossArgs& p, Form f, hipStream_t s) {
  const dim3 grid((unsigned)(p.g.tiles_m * p.g.tiles_n));
  if constexpr (E != 2)
    if (f == kWide) hipLaunchKernelGGL((xent_logits_kernel<Pick<kWide, true, true, E>, BWD>), grid, dim3(256), 0, s, p);
  if (f == kNarrow) hipLaunchKernelGGL((xent_logits_kernel<Pick<kNarrow, true, true, E>, BWD>), grid, dim3(256), 0, s, p);
  if (f == kSlim) hipLaunchKernelGGL((xent_logits_kernel<Pick<kSlim, true, true, E>, BWD>), grid, dim3(256), 0, s, p);
  if constexpr (E == 2)
    if (f == kBlock)
      hipLaunchKernelGGL((xent_logits_kernel<Pick<kBlock, true, true, E>, BWD>), grid, dim3(256), 0, s, p);
  return launch_status("xent_logits_kernel");
}

template <bool A_KC, int E>
int launch_grad(StoreArgs& p, const Way& way, hipStream_t s) {
  const int64_t kt = ceil_div(p.g.K, E == 2 ? kBK32 : kBK16);
  p.g.kt_per_split = (int)std::min(way.range, kt);
  p.g.splits = (int)ceil_div(kt, p.g.kt_per_split);
  const dim3 grid((unsigned)(p.g.tiles_m * p.g.tiles_n * p.g.splits));
  if constexpr (E != 2)
    if (way.form == kWide)
      hipLaunchKernelGGL((xent_grad_kernel<Pick<kWide, A_KC, false, E>>), grid, dim3(256), 0, s, p);
  if (way.form == kNarrow)
    hipLaunchKernelGGL((xent_grad_kernel<Pick<kNarrow, A_KC, false, E>>), grid, dim3(256), 0, s, p);
  if (way.form == kSlim)
    hipLaunchKernelGGL((xent_grad_kernel<Pick<kSlim, A_KC, false, E>>), grid, dim3(256), 0, s, p);
  if constexpr (E == 2)
    if (way.form == kBlock)
      hipLaunchKernelGGL((xent_grad_kernel<Pick<kBlock, A_KC, false, E>>), grid, dim3(256), 0, s, p);
  return launch_status("xent_grad_kernel");
}

int launch_sum(const float* part, int64_t splits, int64_t M, int64_t N, void* c, int64_t ldc, int dtype,
               const float* scale, hipStream_t s) {
  const dim3 grid = strided_grid(M * N / 4);
  const int n = (int)splits, w = (int)N;
  if (dtype == MFX_F32)
    hipLaunchKernelGGL((xent_sum<float>), grid, dim3(256), 0, s, part, n, M, w, static_cast<float*>(c), ldc, scale);
  else if (dtype == MFX_BF16)
    hipLaunchKernelGGL((xent_sum<bf16>), grid, dim3(256), 0, s, part, n, M, w, static_cast<bf16*>(c), ldc, scale);
  else
    hipLaunchKernelGGL((xent_sum<_Float16>), grid, dim3(256), 0, s, part, n, M, w, static_cast<_Float16*>(c), ldc,
                       scale);
  return launch_status("xent_sum");
}

template <int E>
int run_bwd(const mfx_linear_xent_bwd_args& a, const BwdPlan& pl, char* ws, hipStream_t s) {
  float* const scale = E != 2 ? reinterpret_cast<float*>(ws) : nullptr;
  float* const weight = E != 2 ? reinterpret_cast<float*>(ws + 256) : nullptr;
  char* const d = ws + pl.row_bytes;
  float* const dh_part = reinterpret_cast<float*>(d + pl.d_bytes);
  float* const dw_part = reinterpret_cast<float*>(d + pl.d_bytes + pl.dh_bytes);
  const Operand h{a.h, a.h_stride}, dl{d, pl.piece};
  const int t64 = a.target_dtype == MFX_I64, size = dtype_size(a.dtype);
  if (E != 2) {
    hipLaunchKernelGGL(xent_weights, dim3(1), dim3(1024), 0, s, a.dloss, a.targets, t64, (int)a.T, (int)a.V,
                       E == 1 ? 32768.f : 1.f, weight, scale);
    if (int rc = launch_status("xent_weights")) return rc;
  }
  for (int64_t i = 0; i < pl.pieces; ++i) {
    const int64_t v0 = i * pl.piece, nv = std::min(pl.piece, a.V - v0);
    const Operand w{static_cast<const char*>(a.w) + v0 * a.w_stride * size, a.w_stride};
    LossArgs z{};
    const Way zw = choose(E, a.T, nv, a.H, false);
    z.g = shape(h, w, a.T, nv, a.H, E, zw.form);
    z.targets = a.targets;
    z.target64 = t64;
    z.v0 = v0;
    z.V = (int)a.V;
    z.lse = a.lse;
    z.weight = weight ? weight : a.dloss;
    z.d = d;
    z.ldd = pl.piece;
    if (int rc = launch_logits<E, true>(z, zw.form, s)) return rc;
    // (A narrower last piece keeps the first's ways: no more ranges than its.)
    if (a.dw) {
      StoreArgs p{};
      p.g = shape(dl, h, nv, a.H, a.T, E, pl.dw.form);
      p.scale = scale;
      p.c = static_cast<char*>(a.dw) + v0 * a.dw_stride * dtype_size(a.dw_dtype);
      p.ldc = a.dw_stride;
      p.c_f32 = a.dw_dtype == MFX_F32;
      if (pl.dw.ranges > 1) p.part = dw_part;
      if (int rc = launch_grad<false, E>(p, pl.dw, s)) return rc;
      if (p.part)
        if (int rc = launch_sum(dw_part, pl.dw.ranges, nv, a.H, p.c, p.ldc, a.dw_dtype, scale, s)) return rc;
    }
    if (a.dh) {
      StoreArgs p{};
      p.g = shape(dl, w, a.T, a.H, nv, E, pl.dh.form);
      p.scale = scale;
      p.c = a.dh;
      p.ldc = a.dh_stride;
      p.c_f32 = E == 2;
      if (pl.dh_bytes) {
        p.part = dh_part;
        p.add = i > 0;
      }
      if (int rc = launch_grad<true, E>(p, pl.dh, s)) return rc;
    }
  }
  if (a.dh && pl.dh_bytes) return launch_sum(dh_part, pl.dh.ranges, a.T, a.H, a.dh, a.dh_stride, a.dtype, scale, s);
  return MFX_OK;
}

// Forward workspace: the targets' logits, then the partials.
struct FwdPlan {
  Form form;
  int64_t tiles_n;
  size_t row_bytes, part_bytes;
};
FwdPlan plan_fwd(const mfx_linear_xent_args& a) {
  FwdPlan pl{};
  const int E = elem_of(a.dtype);
  pl.form = choose(E, a.T, a.V, a.H, false).form;
  pl.tiles_n = ceil_div(a.V, kFormN[E == 2][pl.form]);
  pl.row_bytes = align256((size_t)a.T * 4);
  pl.part_bytes = align256((size_t)pl.tiles_n * a.T * 4);
  return pl;
}

bool float_dtype(int dt) { return dt == MFX_F32 || dt == MFX_BF16 || dt == MFX_F16; }

// What both directions check; ptrs: every matrix pointer and its row stride.
int check_common(int64_t T, int64_t H, int64_t V, int dtype, int target_dtype) {
  const int64_t lim = 0x7fffffffLL;
  if (T < 0 || H <= 0 || V <= 0) return fail(MFX_E_INVALID, "T must be >= 0, H and V positive");
  if (!float_dtype(dtype)) return fail(MFX_E_UNSUPPORTED, "dtype must be f32, bf16 or f16");
  if (target_dtype != MFX_I32 && target_dtype != MFX_I64)
    return fail(MFX_E_UNSUPPORTED, "target dtype must be i32 or i64");
  if (T > lim - 256 || V > lim - 256 || H > lim - 256) return fail(MFX_E_UNSUPPORTED, "T, H or V too large");
  // (The widest tiles' launches have to fit; `choose` passes over others that do not.)
  const int64_t b = kFormM[first_form(elem_of(dtype))];
  const int64_t t = ceil_div(T, b), v = ceil_div(V, b), k = ceil_div(H, b);
  if (!launch_fits(t * v, 256) || !launch_fits(t * k, 256) || !launch_fits(v * k, 256) ||
      !launch_fits(ceil_div(T, 64), 64 * kCombine))
    return fail(MFX_E_UNSUPPORTED, "problem too large for one launch");
  if (H % (dtype == MFX_F32 ? 4 : 8))
    return fail(MFX_E_UNSUPPORTED, "H must be a multiple of 16 bytes");
  return MFX_OK;
}

int check_matrix(const void* ptr, int64_t stride, int64_t H, int size, const char* what) {
  if (stride < H) return fail(MFX_E_INVALID, std::string(what) + ": row stride must be >= H");
  if ((uintptr_t)ptr % 16 || stride % (16 / size))
    return fail(MFX_E_UNSUPPORTED, std::string(what) + ": rows must be 16-byte aligned");
  if (stride >= kMaxStride) return fail(MFX_E_UNSUPPORTED, std::string(what) + ": row stride too large");
  return MFX_OK;
}

int check_fwd(const mfx_linear_xent_args* a) {
  if (!a) return fail(MFX_E_INVALID, "null args");
  if (int rc = check_common(a->T, a->H, a->V, a->dtype, a->target_dtype)) return rc;
  if (a->T == 0) return MFX_OK;
  if (!a->h || !a->w || !a->targets || !a->loss) return fail(MFX_E_INVALID, "h, w, targets and loss must be non-null");
  const int size = dtype_size(a->dtype);
  if (int rc = check_matrix(a->h, a->h_stride, a->H, size, "h")) return rc;
  return check_matrix(a->w, a->w_stride, a->H, size, "w");
}

int check_bwd(const mfx_linear_xent_bwd_args* a) {
  if (!a) return fail(MFX_E_INVALID, "null args");
  if (int rc = check_common(a->T, a->H, a->V, a->dtype, a->target_dtype)) return rc;
  if (!a->dh && !a->dw) return fail(MFX_E_INVALID, "dh or dw must be non-null");
  if (a->dw && a->dw_dtype != a->dtype && a->dw_dtype != MFX_F32)
    return fail(MFX_E_UNSUPPORTED, "dw dtype must be dtype or f32");
  const int size = dtype_size(a->dtype);
  if (a->dw)
    if (int rc = check_matrix(a->dw, a->dw_stride, a->H, dtype_size(a->dw_dtype), "dw")) return rc;
  if (a->T == 0) return MFX_OK;
  if (!a->h || !a->w || !a->targets || !a->lse || !a->dloss)
    return fail(MFX_E_INVALID, "h, w, targets, lse and dloss must be non-null");
  if (int rc = check_matrix(a->h, a->h_stride, a->H, size, "h")) return rc;
  if (int rc = check_matrix(a->w, a->w_stride, a->H, size, "w")) return rc;
  if (a->dh) return check_matrix(a->dh, a->dh_stride, a->H, size, "dh");
  return MFX_OK;
}

// The caller's workspace or the library's scratch for the stream.
int take_workspace(void* given, size_t given_bytes, size_t need, const char* query, hipStream_t s, char** out) {
  if (given) {
    if (given_bytes < need) return fail(MFX_E_WORKSPACE, std::string("workspace smaller than ") + query + "()");
    if ((uintptr_t)given % 256) return fail(MFX_E_INVALID, "workspace must be 256-byte aligned");
    *out = static_cast<char*>(given);
    return MFX_OK;
  }
  *out = static_cast<char*>(device_scratch(need, s));
  return *out ? MFX_OK : MFX_E_HIP;
}

// dw of no rows.
template <typename T>
__global__ __launch_bounds__(256) void xent_zero(T* c, int64_t rows, int64_t n, int64_t ldc) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * n; i += (int64_t)gridDim.x * 256)
    c[i / n * ldc + i % n] = from_f32<T>(0.f);
}

}  // namespace
}  // namespace xent
}  // namespace mfx

extern "C" {

size_t mfx_linear_xent_workspace_size(const mfx_linear_xent_args* args) {
  using namespace mfx::xent;
  if (check_fwd(args) != MFX_OK || args->T == 0) return 0;
  const FwdPlan pl = plan_fwd(*args);
  return pl.row_bytes + 2 * pl.part_bytes;
}

int mfx_linear_xent(const mfx_linear_xent_args* args, void* stream) {
  using namespace mfx;
  using namespace mfx::xent;
  if (int rc = check_fwd(args)) return rc;
  if (args->T == 0) return MFX_OK;
  const mfx_linear_xent_args& a = *args;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const FwdPlan pl = plan_fwd(a);
  char* ws = nullptr;
  if (int rc = take_workspace(a.workspace, a.workspace_bytes, pl.row_bytes + 2 * pl.part_bytes,
                              "mfx_linear_xent_workspace_size", s, &ws))
    return rc;
  LossArgs z{};
  z.g = shape(Operand{a.h, a.h_stride}, Operand{a.w, a.w_stride}, a.T, a.V, a.H, elem_of(a.dtype),
              pl.form);
  z.targets = a.targets;
  z.target64 = a.target_dtype == MFX_I64;
  z.V = (int)a.V;
  z.picked = reinterpret_cast<float*>(ws);
  z.part_m = reinterpret_cast<float*>(ws + pl.row_bytes);
  z.part_l = reinterpret_cast<float*>(ws + pl.row_bytes + pl.part_bytes);
  int rc;
  if (a.dtype == MFX_F32) rc = launch_logits<2, false>(z, pl.form, s);
  else if (a.dtype == MFX_F16) rc = launch_logits<1, false>(z, pl.form, s);
  else rc = launch_logits<0, false>(z, pl.form, s);
  if (rc) return rc;
  hipLaunchKernelGGL(xent_combine, dim3((unsigned)ceil_div(a.T, 64)), dim3(64 * kCombine), 0, s, z.part_m, z.part_l, z.picked,
                     a.targets, z.target64, (int)a.T, (int)a.V, (int)pl.tiles_n, a.loss, a.lse);
  return launch_status("xent_combine");
}

size_t mfx_linear_xent_bwd_workspace_size(const mfx_linear_xent_bwd_args* args) {
  using namespace mfx::xent;
  if (check_bwd(args) != MFX_OK || args->T == 0) return 0;
  return plan_bwd(*args).total;
}

int mfx_linear_xent_bwd(const mfx_linear_xent_bwd_args* args, void* stream) {
  using namespace mfx;
  using namespace mfx::xent;
  if (int rc = check_bwd(args)) return rc;
  const mfx_linear_xent_bwd_args& a = *args;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a.T == 0) {
    if (!a.dw) return MFX_OK;
    const dim3 grid = strided_grid(a.V * a.H);
    if (a.dw_dtype == MFX_F32)
      hipLaunchKernelGGL((xent_zero<float>), grid, dim3(256), 0, s, static_cast<float*>(a.dw), a.V, a.H, a.dw_stride);
    else  // (zero has the same bits in both 16-bit types)
      hipLaunchKernelGGL((xent_zero<bf16>), grid, dim3(256), 0, s, static_cast<bf16*>(a.dw), a.V, a.H, a.dw_stride);
    return launch_status("xent_zero");
  }
  const BwdPlan pl = plan_bwd(a);
  char* ws = nullptr;
  if (int rc = take_workspace(a.workspace, a.workspace_bytes, pl.total, "mfx_linear_xent_bwd_workspace_size", s, &ws))
    return rc;
  if (a.dtype == MFX_F32) return run_bwd<2>(a, pl, ws, s);
  return a.dtype == MFX_F16 ? run_bwd<1>(a, pl, ws, s) : run_bwd<0>(a, pl, ws, s);
}

}  // extern "C"

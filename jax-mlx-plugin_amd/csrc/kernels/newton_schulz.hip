// Matrices orthogonalised by Newton-Schulz products, and the weight update
// built on them (no counterpart in the reference):
//
//   X = U / (|U|_F + eps),   `steps` times:  X = (a I + b A + c A^2) X,  A = X X^T
//
// A is taken of the smaller side: for a matrix taller than wide A = X^T X and X =
// X (a I + b A + c A^2), the same products with the operands' roles changed, no
// transpose stored.  Each step is three products on the matrix cores:
//
//   gram     A = X X^T           symmetric
//   square   Q = a I + b A + c A A   symmetric (A is: both operands are A's rows)
//   apply    X = Q X   or   X Q
//
// of 2 s^2 l, 2 s^3 and 2 s^2 l operations (s, l the sides); gram and square form
// only the tiles on and below the diagonal and store each twice.
//
// Where X is long (3 small products take less than gram and apply) two steps are
// taken at once: A of the second is Q A Q, since Q is a polynomial in A, and X is
// multiplied by Q' Q, so gram and apply run every other step:
//
//   T = Q A,  A' = T Q,  Q' = a I + b A' + c A' A',  P = Q' Q,  X = P X
//
// all of them symmetric.  Their entries are off by as much as before (1.7e-6 to
// 2.1e-6 in fp32, 4e-6 with a few large directions), but in one f16 term by up to
// three times, so it is for two terms.
//
// Precision.  The products' operands are f16, in one term or in two (a leading
// one and what it leaves out: 22 bits, three products for one, pair_gemm16.h), all
// sums fp32.  X, A and Q are stored times powers of two that the host derives from
// the bound that the coefficients give their norms, so that no entry overflows
// and the second terms stay clear of the smallest f16.  A singular value that
// is small beside |U| is raised by up to a^steps (485), and with it what the
// roundings put there.  Measured against 64 bits, 512 x 512 whose entries are one
// direction and noise of 1, 1/100 and 1/300 of its size: off by 1.5e-6, 1.7e-5 and
// 4.5e-5 of the result's norm in two terms, products of fp32 matrices by 2.2e-6, 2.4e-5 and
// 6.7e-5; in one term by 1.3e-3, 2.1e-2 and 5.8e-2, more than any result's own rounding
// (bf16 1.7e-3).  So two terms are the rule, whatever the types, and one term is for
// callers who ask for it and know their gradients.  The norm is summed
// in 64 bits (squares of small gradients leave the range of fp32).
//
// What bounds it.  Large products: what the L2s deliver to LDS, 7 to 8 TB/s in
// tiles of 192 and 256 (4096 a side: 199 us gram, 211 square, 327 apply, whose three
// products of f16 run at a library product's 1.26 PFLOP/s; in one term 87, 92 and 122).  2048 a
// side 36 to 38 us and a join of 10 to 12.  Small ones: 512 a side 9 to 12 us, half of it a start and an end.
// Together, five steps: 512 x 512 158 us, 12 of 2048 x 512 in bf16 429 to 447, the update of
// 2048 x 8200 in f32 1.57 to 1.64 ms, of 4096 x 4096 in bf16 3.70 to 3.74.
//
// The update takes its momentum on the way in (ns_norm, ns_split) and adds to the
// weights in the last product's epilogue.
#include <algorithm>
#include <cmath>

#include "rowvec.h"
#include "workspace.h"
#include "pair_gemm16.h"

namespace mfx {
namespace ns {
namespace {

using namespace xent;
using rowvec::load_run;
using rowvec::store_run;

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ---- the matrix on its way in ------------------------------------------------------

struct InArgs {
  const void* g;
  const void* buf;     // momentum (null: none)
  void* buf_out;
  double* norm;        // [B][parts] sums of squares
  uint16_t* x;         // [B][m][ld] leading terms (f16), the second `lo` elements behind
  int64_t gs_b, gs_r, bs_b, bs_r, os_b, os_r, lo;
  int m, n, ld, parts, two;
  int g_dt, buf_dt;
  float mu, eps, scale;  // scale: the power of two that X is stored at
  int nesterov;
};

__device__ __forceinline__ void load8(const void* p, int dt, int64_t at, int e, int n, float (&out)[8]) {
  if (dt == MFX_F32) load_run<float, 8>(static_cast<const float*>(p) + at, e, n, 0.f, out);
  else if (dt == MFX_BF16) load_run<bf16, 8>(static_cast<const bf16*>(p) + at, e, n, 0.f, out);
  else load_run<_Float16, 8>(static_cast<const _Float16*>(p) + at, e, n, 0.f, out);
}

__device__ __forceinline__ void store8(void* p, int dt, int64_t at, int e, int n, const float (&v)[8]) {
  if (dt == MFX_F32) store_run<float, 8>(static_cast<float*>(p) + at, e, n, v);
  else if (dt == MFX_BF16) store_run<bf16, 8>(static_cast<bf16*>(p) + at, e, n, v);
  else store_run<_Float16, 8>(static_cast<_Float16*>(p) + at, e, n, v);
}

// The chunk's U, and in `b` the new momentum.
__device__ __forceinline__ void take(const InArgs& a, int64_t bz, int row, int e, float (&u)[8], float (&b)[8]) {
  load8(a.g, a.g_dt, bz * a.gs_b + row * a.gs_r, e, a.n, u);
  if (!a.buf) return;
  load8(a.buf, a.buf_dt, bz * a.bs_b + row * a.bs_r, e, a.n, b);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    b[j] = fmaf(a.mu, b[j], (1.f - a.mu) * u[j]);
    u[j] = a.nesterov ? fmaf(a.mu, b[j], (1.f - a.mu) * u[j]) : b[j];
  }
}

__device__ __forceinline__ double block_sum(double v, double* lds) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

// Sums of squares: workgroup (part, matrix).
__global__ __launch_bounds__(256) void ns_norm(InArgs a) {
  __shared__ double lds[4];
  const uint32_t cpr = (uint32_t)a.ld / 8, units = (uint32_t)a.m * cpr;
  double s = 0.0;
  for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < units; i += a.parts * 256) {
    const uint32_t row = i / cpr;
    float u[8], b[8];
    take(a, blockIdx.y, (int)row, (int)(i - row * cpr) * 8, u, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) s = fma((double)u[j], (double)u[j], s);
  }
  s = block_sum(s, lds);
  if (threadIdx.x == 0) a.norm[(int64_t)blockIdx.y * a.parts + blockIdx.x] = s;
}

// What the leading f16 term of x leaves out.
__device__ __forceinline__ float rest(float x) { return x - (float)static_cast<f16>(x); }

// X = U / (|U| + eps), and the momentum.
__global__ __launch_bounds__(256) void ns_split(InArgs a) {
  __shared__ double lds[4];
  double sum = 0.0;  // (the same order in every workgroup)
  for (int i = threadIdx.x; i < a.parts; i += 256) sum += a.norm[(int64_t)blockIdx.y * a.parts + i];
  sum = block_sum(sum, lds);
  // (In 64 bits: the factor of matrices smaller than 1e-34 is past fp32's range.)
  const double f = (double)a.scale / (sqrt(sum) + (double)a.eps);
  const uint32_t cpr = (uint32_t)a.ld / 8, units = (uint32_t)a.m * cpr;
  uint16_t* const x = a.x + (int64_t)blockIdx.y * a.m * a.ld;
  for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < units; i += gridDim.x * 256) {
    const uint32_t row = i / cpr;
    const int e = (int)(i - row * cpr) * 8;
    float u[8], b[8];
    take(a, blockIdx.y, (int)row, e, u, b);
    if (a.buf) store8(a.buf_out, a.buf_dt, (int64_t)blockIdx.y * a.os_b + row * a.os_r, e, a.n, b);
    // (Zeros in the columns past n: 0 times a factor that may be infinite would not be.)
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = e + j < a.n ? (float)((double)u[j] * f) : 0.f;
    *reinterpret_cast<uint4*>(x + (int64_t)i * 8) = rowvec::pack16<_Float16>(u);
    if (!a.two) continue;
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = rest(u[j]);
    *reinterpret_cast<uint4*>(x + a.lo + (int64_t)i * 8) = rowvec::pack16<_Float16>(u);
  }
}

// ---- the products ------------------------------------------------------------------

enum Mode { kGram, kSquare, kApply };

// The forms of a product's tiles: square ones, since a symmetric product's
// tiles are stored transposed too.
// kMid is for operands along k.  In one term it is for symmetric products of about 4096 a
// side, 253 tiles of 192 x 192 where 136 of 256 x 256 leave half the CUs without one: 81
// and 87 us (gram, square; by themselves, over and over) for 89 and 100, or 94 and 97 in 128 x 128.  In two terms the
// products of 32 k with their reads from LDS fit in registers, those of 256 x 256 do
// not: 187 and 202 us for 258 and 264 (4096 a side), 42 and 45 for 52 and 55 (2048).
enum Form { kWide, kNarrow, kSlim, kMid };
constexpr int kForms = 4, kSide[kForms] = {256, 128, 64, 192};

// k of a tile: 32, but of two terms in the two larger of the first forms 16 (their
// stages, and the fragments of more, would not fit).
constexpr int depth(Form f, bool two) { return two && f < kSlim ? 16 : 32; }

template <int SIDE, bool A_KC, bool B_KC, bool P>
struct Cfg : Config<SIDE, SIDE, SIDE == 64 ? 1 : 2, 2, A_KC, B_KC, 1> {
  static constexpr bool PAIR = P;  // operands in two terms
  static constexpr bool ROT = false;
  static constexpr int WAVES = SIDE == 256 || SIDE == 192 ? 1 : SIDE == 128 ? 2 : 3;  // per SIMD
  static constexpr int BK = depth(SIDE == 64 ? kSlim : SIDE == 192 ? kMid : kWide, P);
  static constexpr int STAGES = SIDE == 192 && P ? 2 : 4;  // (its 54 products of a tile cover taking up the next)
  static constexpr int SMEM = STAGES * 4 * SIDE * BK * (1 + P);
};

struct ProdArgs {
  GemmShape g;          // of one matrix; tiles_m x tiles_n tiles (symmetric: the lower triangle)
  int64_t as, bs;       // elements from matrix to matrix of the operands
  int64_t tiles, all;   // tiles of a matrix and of all
  int kt;               // k-tiles of a tile
  int symmetric, two;
  // Whole tiles first, a workgroup each; then of each other tile `splits` ranges of
  // `per` k-tiles, which leave partial sums.
  int64_t whole;
  int splits, per;
  float* part;          // [splits][tiles split][NT * FM * FN * 16]
  float c1, c2, c3;     // gram, apply: c1 C;  square: c1 C + c2 A + c3 I
  // Result in f16 terms ...
  uint16_t* c;          // [rows][ldc]
  int64_t ldc, cs, lo;
  // ... or, at the end, the result or the updated weights
  void* out;            // null: terms
  const void* w;        // out = keep w + c1 C
  int64_t os_b, os_r, ws_b, ws_r;
  int out_dt;
  float keep;
};

// Tile t of a matrix, in bands of 8 tile rows (of 4 where only the lower triangle
// is there) walked column by column, so that the tiles at work on an XCD share
// operand panels in its L2.
__device__ __forceinline__ void tile_of(const ProdArgs& p, int t, int& tm, int& tn) {
  if (!p.symmetric) {
    const int band = 8 * p.g.tiles_n, b = t / band, rows = min(8, p.g.tiles_m - b * 8);
    t -= b * band;
    tm = b * 8 + t % rows;
    tn = t / rows;
    return;
  }
  int r0 = 0, rows;
  for (;; r0 += 4) {
    rows = min(4, p.g.tiles_m - r0);
    const int n = rows * r0 + rows * (rows + 1) / 2;
    if (t < n) break;
    t -= n;
  }
  if (t < rows * r0) {
    tm = r0 + t % rows;
    tn = t / rows;
    return;
  }
  // The band's own triangle.
  t -= rows * r0;
  int c = 0;
  while (t >= rows - c) t -= rows - c++;
  tm = r0 + c + t;
  tn = r0 + c;
}

// What becomes of a block of sums, rows m0 .. + 31 by columns n0 .. + FN * 32 of
// matrix bz, by one wavefront.  The sums go to LDS (st: FN * 4 KB of the
// wavefront's own), chunk c (four) of row r at slot c ^ (r % chunks) (of 24 chunks: % 8), and from there in
// runs of eight along a row; of a symmetric product's tile off the diagonal
// (`turned`) the values go back there and out once more in runs of eight down a
// column, which are a row's of the other half.
template <int FN, Mode MODE>
__device__ __forceinline__ void finish_rows(const ProdArgs& p, int64_t bz, int m0, int n0, bool turned, float* st,
                                            const f32x16 (&acc)[FN]) {
  constexpr int W = FN * 32, QUADS = W / 4, TURN = QUADS & (QUADS - 1) ? 7 : QUADS - 1;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int M = p.g.M, N = p.g.N;
  {
    int l = lane & 31;  // (opaque: no address is kept through the products)
    asm volatile("" : "+v"(l));
    f32x4* const row = reinterpret_cast<f32x4*>(st + l * W);
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        row[(j * 8 + g * 2 + half) ^ (l & TURN)] =
            f32x4{acc[j][g * 4], acc[j][g * 4 + 1], acc[j][g * 4 + 2], acc[j][g * 4 + 3]};
  }
  fence();
  constexpr int RUNS = FN * 4, STEPS = RUNS / 2;  // of a row; steps of 64 runs
  uint16_t* const c = p.c + bz * p.cs;
  // One or two f16 terms of a run.
  auto put = [&](int64_t at, const float (&v)[8]) __attribute__((always_inline)) {
    *reinterpret_cast<uint4*>(c + at) = rowvec::pack16<_Float16>(v);
    if (p.two) {
      float r[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] = rest(v[e]);
      *reinterpret_cast<uint4*>(c + p.lo + at) = rowvec::pack16<_Float16>(r);
    }
  };
  // (Unrolled for a square product's reads of A to overlap; the last product's
  // end, of any type and alignment, stays a loop.)
  constexpr int UNROLL = MODE == kSquare ? STEPS : 2;
#pragma unroll UNROLL
  for (int k = 0; k < STEPS; ++k) {
    const int at = k * 64 + lane, r = at / RUNS, run = at % RUNS, m = m0 + r, n = n0 + run * 8;
    if (m >= M || n >= N) continue;
    f32x4* const row = reinterpret_cast<f32x4*>(st + r * W);
    f32x4 &x = row[(run * 2) ^ (r & TURN)], &y = row[(run * 2 + 1) ^ (r & TURN)];
    float v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= p.c1;
    if (MODE == kApply && p.out) {
      if (p.w) {
        float w[8];
        load8(p.w, p.out_dt, bz * p.ws_b + m * p.ws_r, n, N, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fmaf(p.keep, w[e], v[e]);
      }
      store8(p.out, p.out_dt, bz * p.os_b + m * p.os_r, n, N, v);
      continue;
    }
    if constexpr (MODE == kSquare) {  // a I + b A (A's rows are padded to whole runs)
      const uint16_t* from = static_cast<const uint16_t*>(p.g.a.p) + bz * p.as + (int64_t)m * p.g.a.ld + n;
      float a[8];
      rowvec::unpack16<_Float16>(*reinterpret_cast<const uint4*>(from), a);
      if (p.two) {
        float b[8];
        rowvec::unpack16<_Float16>(*reinterpret_cast<const uint4*>(from + p.g.a.lo), b);
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] += b[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = fmaf(p.c2, a[e], v[e]) + (m == n + e ? p.c3 : 0.f);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = n + e < N ? v[e] : 0.f;  // (zeros in the padding)
    if (MODE != kApply && turned) {
      x = f32x4{v[0], v[1], v[2], v[3]};
      y = f32x4{v[4], v[5], v[6], v[7]};
    }
    put((int64_t)m * p.ldc + n, v);
  }
  if (MODE == kApply || !turned) return;
  fence();
#pragma unroll 2
  for (int k = 0; k < W; k += 16) {
    const int r = k + lane / 4, run = lane % 4, n = n0 + r, m = m0 + run * 8;
    if (n >= N || m >= M) continue;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int row = run * 8 + e;
      v[e] = st[row * W + ((r >> 2) ^ (row & TURN)) * 4 + (r & 3)];
    }
    // (Nothing went over rows past the matrix, which hold sums of what lies there.)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = m + e < M ? v[e] : 0.f;
    put((int64_t)n * p.ldc + m, v);
  }
}

// What becomes of a tile's sums: a wavefront goes through its block 32 rows at a
// time, with fences between, so that no more than one set of values and addresses is
// live beside the sums.
template <class C, Mode MODE>
__device__ __forceinline__ void finish(const ProdArgs& p, int64_t bz, int tm, int tn, char* smem, Acc<C>& acc) {
  constexpr int FM = C::FM, FN = C::FN;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % C::WM, wn = wave / C::WM;
  static_assert(FN * 4096 <= C::SMEM / C::NW, "a wavefront's part of the stages, which are free");
  float* const st = reinterpret_cast<float*>(smem + wave * (C::SMEM / C::NW));
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    f32x16 rows[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) rows[j] = acc[j][i];
    finish_rows<FN, MODE>(p, bz, tm * C::BM + (wm * FM + i) * 32, tn * C::BN + wn * FN * 32, MODE != kApply && tm != tn,
                          st, rows);
    fence();
  }
}

// This workgroup's place among `n`, dealt to the 8 XCDs in turn: each takes a
// run of neighbours, which share operand panels in its L2.
__device__ __forceinline__ int64_t dealt(int64_t id, int64_t n) {
  const int64_t per = n >> 3, rest = n & 7, xcd = id & 7;
  return (id >> 3) + xcd * per + min(xcd, rest);
}

template <class C, Mode MODE>
__global__ __launch_bounds__(C::NT, C::WAVES) void ns_product(ProdArgs p) {
  __shared__ __attribute__((aligned(16))) char smem[C::SMEM];
  constexpr int PART = C::NT * C::FM * C::FN * 16;
  int64_t tile, slot = -1;
  int kt0 = 0, kt1 = p.kt;
  if ((int64_t)blockIdx.x < p.whole) {
    tile = dealt(blockIdx.x, p.whole);
  } else {
    // (Range by range: workgroups next to each other read the same k of neighbouring
    // tiles.  Tile by tile each would read a range of its own, 200 us for
    // 130 where 36 tiles are split into 7.)
    const int64_t rest = p.all - p.whole;
    slot = dealt(blockIdx.x - p.whole, rest * p.splits);
    const int split = (int)(slot / rest);
    tile = p.whole + (slot - split * rest);
    kt0 = split * p.per;
    kt1 = min(kt1, kt0 + p.per);
  }
  const int bz = (int)(tile / p.tiles);
  int tm, tn;
  tile_of(p, (int)(tile - (int64_t)bz * p.tiles), tm, tn);
  GemmShape g = p.g;
  g.a.p = static_cast<const uint16_t*>(g.a.p) + bz * p.as;
  g.b.p = static_cast<const uint16_t*>(g.b.p) + bz * p.bs;
  Acc<C> acc;
  bf16* const stages = reinterpret_cast<bf16*>(smem);
  if constexpr (C::PAIR && C::BK == 32)
    gemm_pair16_flat<C>(g, tm * C::BM, tn * C::BN, kt0, kt1, stages, acc);
  else if constexpr (C::PAIR) gemm_pair16<C>(g, tm * C::BM, tn * C::BN, kt0, kt1, stages, acc);
  else gemm_tile16<C>(g, tm * C::BM, tn * C::BN, kt0, kt1, stages, acc);
  __syncthreads();  // the stages are free
  if (slot < 0) {
    finish<C, MODE>(p, bz, tm, tn, smem, acc);
    return;
  }
  uint32_t tid = threadIdx.x;  // (opaque: no address is kept through the products)
  asm volatile("" : "+v"(tid));
  f32x4* const to = reinterpret_cast<f32x4*>(p.part + slot * PART) + tid;
#pragma unroll
  for (int j = 0; j < C::FN; ++j)
#pragma unroll
    for (int i = 0; i < C::FM; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        to[((j * C::FM + i) * 4 + q) * C::NT] =
            f32x4{acc[j][i][q * 4], acc[j][i][q * 4 + 1], acc[j][i][q * 4 + 2], acc[j][i][q * 4 + 3]};
}

// The split tiles: their partial sums in order, then what finish_rows does, each
// 32 x 32 block by a wavefront of its own (few tiles are split into many
// ranges: a workgroup a tile took 270 us over 8 tiles of 16).
constexpr int kJoinWaves = 4;
template <class C, Mode MODE>
__global__ __launch_bounds__(kJoinWaves * 64) void ns_join(ProdArgs p) {
  constexpr int PART = C::NT * C::FM * C::FN * 16, BLOCKS = C::NW * C::FM * C::FN;
  static_assert(BLOCKS % kJoinWaves == 0, "a workgroup's blocks are of one tile");
  __shared__ __attribute__((aligned(16))) float st[kJoinWaves][1024];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t id = (int64_t)blockIdx.x * kJoinWaves + wave, tile = id / BLOCKS, rest = p.all - p.whole;
  const int block = (int)(id - tile * BLOCKS), of = block / (C::FM * C::FN), ij = block % (C::FM * C::FN);
  const int i = ij % C::FM, j = ij / C::FM, wm = of % C::WM, wn = of / C::WM;
  const float* const part = p.part + tile * PART + ij * (C::NT * 16) + (of * 64 + lane) * 4;
  f32x16 acc[1];
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[0][e] = 0.f;
  constexpr int U = 4;  // partials in flight
  for (int k = 0; k < p.splits; k += U) {
    f32x4 v[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int q = 0; q < 4; ++q)  // (past the last: the last again, not added)
        v[u][q] = *reinterpret_cast<const f32x4*>(part + min(k + u, p.splits - 1) * rest * PART + q * (C::NT * 4));
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k + u < p.splits)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[0][e] += v[u][e / 4][e % 4];
  }
  const int64_t t = p.whole + tile, bz = t / p.tiles;
  int tm, tn;
  tile_of(p, (int)(t - bz * p.tiles), tm, tn);
  finish_rows<1, MODE>(p, bz, tm * C::BM + (wm * C::FM + i) * 32, tn * C::BN + (wn * C::FN + j) * 32,
                       MODE != kApply && tm != tn, st[wave], acc);
}

// ---- host ------------------------------------------------------------------------

bool float_dtype(int dt) { return dt == MFX_F32 || dt == MFX_BF16 || dt == MFX_F16; }

constexpr int64_t kMaxSide = int64_t(1) << 20;  // rows of a tile are addressed within 31 bits
constexpr int kMaxSteps = 32;

// How a product's tiles are shared out.
struct Way {
  Form form;
  int64_t tiles, whole;  // of all matrices; those that are not split
  int splits, per;
  float us;
};

// Microseconds of a k-tile with `slots` workgroups on each CU (`alone` of that
// with none), once for each round of workgroups and more of it for a square
// product's reads of A, and of a join: once, and by its partial sums at `rate`
// TB/s.  Fitted to the kernels' times over 13 shapes from [128, 512] to [4096, 4096]
// and 12 of [512, 2048], each product in every form with 1 to 12 ranges.
struct Cost {
  int slots;
  float kt, alone, each, square, join, rate;
};
constexpr Cost kCost[2][kForms] = {{{1, 0.818f, 0.73f, 12.4f, 6.5f, 1.7f, 9.9f},
                               {2, 0.597f, 0.01f, 3.9f, 1.9f, 6.9f, 12.9f},
                               {4, 0.536f, 0.09f, 3.6f, 1.3f, 7.3f, 60.f},
                               {1, 0.639f, 0.71f, 5.9f, 5.9f, 8.3f, 26.f}},
                              {{1, 1.240f, 0.69f, 10.0f, 13.2f, 2.8f, 8.3f},
                               {2, 0.947f, 0.00f, 1.8f, 4.5f, 8.0f, 8.7f},
                               {2, 0.578f, 0.18f, 3.4f, 1.9f, 7.6f, 60.f},
                              {1, 1.494f, 0.74f, 7.4f, 9.1f, 4.6f, 12.9f}}};

// Of `wgs` workgroups of `n` k-tiles each.
float rounds_us(const Cost& c, int64_t wgs, int64_t n, bool square) {
  const int64_t cus = device_cu_count(), slots = c.slots * cus, rest = wgs % slots;
  const float once = c.each + (square ? c.square : 0.f);
  float t = (float)(wgs / slots) * ((float)n * c.kt + once);
  if (rest) {
    const float load = c.slots == 1 ? (float)rest / (float)cus : (float)ceil_div(rest, cus) / (float)c.slots;
    t += (float)n * c.kt * (c.alone + (1.f - c.alone) * load) + once;
  }
  return t;
}

// The way that takes least by these: every form, its tiles whole or those of the
// last, partly filled round split along k into ranges of at least 8 k-tiles.
// along: both operands are rows along k.
Way choose(int64_t B, int64_t M, int64_t N, int64_t K, Mode mode, bool two, bool along) {
  const int64_t cus = device_cu_count();
  Way best{};
  float least = INFINITY;
  for (int f = kWide; f < kForms; ++f) {
    if (f == kMid && !along) continue;
    const Cost& c = kCost[two][f];
    const int64_t side = kSide[f], tm = ceil_div(M, side), tn = ceil_div(N, side), kt = ceil_div(K, depth((Form)f, two));
    const int64_t tiles = B * (mode != kApply ? tm * (tm + 1) / 2 : tm * tn), rest = tiles % (c.slots * cus);
    if (!launch_fits(tiles, 256)) continue;
    const float whole = rounds_us(c, tiles, kt, mode == kSquare);
    if (whole < least) {
      least = whole;
      best = Way{(Form)f, tiles, tiles, 0, 0, whole};
    }
    for (int64_t n = 2; rest && n <= 64 && n * 8 <= kt; ++n) {
      const int64_t per = ceil_div(kt, n), wgs = rest * n;
      if (ceil_div(kt, per) != n || !launch_fits(tiles - rest + wgs, 256)) continue;
      const float t = rounds_us(c, tiles - rest, kt, mode == kSquare) + rounds_us(c, wgs, per, false) + c.join +
                      (float)wgs * (float)(side * side) * 8e-6f / c.rate;
      if (t < least) {
        least = t;
        best = Way{(Form)f, tiles, tiles - rest, (int)n, (int)per, t};
      }
    }
  }
  return best;
}

size_t part_bytes(const Way& w) {
  return (size_t)w.splits * (w.tiles - w.whole) * kSide[w.form] * kSide[w.form] * 4;
}

struct Plan {
  int64_t B, m, n, s, l, ld, lds;  // the matrix, its smaller and larger side, rows of X and of A
  bool wide;
  int two, steps, parts;
  bool paired;
  Way gram, square, apply, small;  // small: of two matrices of the smaller side
  size_t norm_bytes, x_bytes, a_bytes, part, total;
  // The powers of two that X, A, Q are stored at, and of two steps taken together Q A and Q' Q.
  float ex[kMaxSteps + 1], ea[kMaxSteps], eq[kMaxSteps], et[kMaxSteps], ep[kMaxSteps];
};

// The largest power of two that keeps values up to `most` within f16.
float fit(double most) { return (float)std::exp2(std::floor(std::log2(60000.0 / most))); }

// Bounds of the iterates' norms: X starts at 1 or less; over the spectrum [0, u]
// of X the polynomials' largest values are at its end or where a derivative is 0.
int plan_scales(Plan& pl, const float* coeffs, int num) {
  double u = 1.0, before = 1.0;
  for (int i = 0; i < pl.steps; ++i) {
    const float* k = coeffs + 3 * (num == 1 ? 0 : i);
    const double a = k[0], b = k[1], c = k[2];
    if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return fail(MFX_E_INVALID, "coefficients must be finite");
    u *= 1.01;  // (what rounding adds)
    const double top = u * u;
    auto q = [&](double s) { return std::fabs(a + b * s + c * s * s); };
    double qm = std::max(q(0.0), q(top));
    if (c != 0.0) {
      const double s = -b / (2.0 * c);
      if (s > 0.0 && s < top) qm = std::max(qm, q(s));
    }
    double next = std::sqrt(top) * q(top);
    auto visit = [&](double s) {
      if (s > 0.0 && s < top) next = std::max(next, std::sqrt(s) * q(s));
    };
    // d/dx of x (a + b x^2 + c x^4) is 0 at a + 3 b s + 5 c s^2 = 0.
    if (c != 0.0) {
      const double d = 9.0 * b * b - 20.0 * a * c;
      if (d >= 0.0) {
        visit((-3.0 * b + std::sqrt(d)) / (10.0 * c));
        visit((-3.0 * b - std::sqrt(d)) / (10.0 * c));
      }
    } else if (b != 0.0) {
      visit(-a / (3.0 * b));
    }
    if (!(qm <= 256.0) || !(next <= 16.0))
      return fail(MFX_E_UNSUPPORTED, "the coefficients let the iteration grow too large");
    pl.ex[i] = fit(u);
    pl.ea[i] = fit(top);
    qm = std::max(qm, 1.0 / 256.0);
    pl.eq[i] = fit(qm);
    pl.et[i] = fit(1.02 * qm * top);
    if (i) pl.ep[i - 1] = fit(1.02 * before * qm);
    before = qm;
    u = std::max(next, 1.0 / 16.0);
  }
  pl.ex[pl.steps] = 1.f;  // (the result is not stored in terms)
  return MFX_OK;
}

int plan_common(Plan& pl, int64_t B, int64_t m, int64_t n, int64_t steps, const float* coeffs, int num_coeffs, float eps,
                int terms) {
  if (B < 0 || m <= 0 || n <= 0) return fail(MFX_E_INVALID, "batch must be >= 0, m and n positive");
  if (steps < 1 || !coeffs || (num_coeffs != 1 && num_coeffs != steps))
    return fail(MFX_E_INVALID, "steps must be >= 1, coefficients for all steps or for each");
  if (steps > kMaxSteps) return fail(MFX_E_UNSUPPORTED, "more than 32 steps are not supported");
  if (!(eps >= 0.f) || !std::isfinite(eps)) return fail(MFX_E_INVALID, "eps must be finite and >= 0");
  if (terms < 0 || terms > 2) return fail(MFX_E_INVALID, "terms must be 0, 1 or 2");
  if (m > kMaxSide || n > kMaxSide || m * ceil_div(n, 8) > 0x7fffffffLL - 0x1000000 || B > 65535)
    return fail(MFX_E_UNSUPPORTED, "problem too large for one launch");
  pl.B = B, pl.m = m, pl.n = n;
  pl.wide = m <= n;
  pl.s = std::min(m, n), pl.l = std::max(m, n);
  pl.ld = ceil_div(n, 8) * 8;
  pl.lds = ceil_div(pl.s, 8) * 8;
  pl.steps = (int)steps;
  pl.two = terms != 1;
  if (int rc = plan_scales(pl, coeffs, num_coeffs)) return rc;
  if (B == 0) return MFX_OK;
  pl.gram = choose(B, pl.s, pl.s, pl.l, kGram, pl.two, pl.wide);
  pl.square = choose(B, pl.s, pl.s, pl.s, kSquare, pl.two, true);
  pl.apply = choose(B, m, n, pl.s, kApply, pl.two, !pl.wide);
  if (!pl.gram.tiles || !pl.square.tiles || !pl.apply.tiles)
    return fail(MFX_E_UNSUPPORTED, "problem too large for one launch");
  if (pl.two) {
    pl.small = choose(B, pl.s, pl.s, pl.s, kGram, true, true);
    pl.paired = pl.steps > 1 && pl.small.tiles && 3.f * pl.small.us < pl.gram.us + pl.apply.us;
  }
  if (!launch_fits(B * std::min<int64_t>(2048, ceil_div(m * (pl.ld / 8), 256)), 256))
    return fail(MFX_E_UNSUPPORTED, "problem too large for one launch");
  // Parts of a matrix's sum of squares: of 512 chunks or more, at most four a thread of ns_split.
  pl.parts = (int)std::min<int64_t>(1024, ceil_div(m * (pl.ld / 8), 512));
  pl.norm_bytes = align256((size_t)B * pl.parts * 8);
  pl.x_bytes = align256((size_t)B * m * pl.ld * 2 * (1 + pl.two));
  pl.a_bytes = align256((size_t)B * pl.s * pl.lds * 2 * (1 + pl.two));
  pl.part = align256(std::max(std::max(part_bytes(pl.gram), part_bytes(pl.square)),
                              std::max(part_bytes(pl.apply), pl.paired ? part_bytes(pl.small) : 0)));
  pl.total = pl.norm_bytes + 2 * pl.x_bytes + (2 + pl.paired) * pl.a_bytes + pl.part;
  return MFX_OK;
}

template <class C, Mode MODE>
int launch(const ProdArgs& p, hipStream_t s) {
  hipLaunchKernelGGL((ns_product<C, MODE>), dim3((unsigned)(p.whole + p.splits * (p.all - p.whole))), dim3(C::NT), 0, s, p);
  return launch_status("ns_product");
}

template <int SIDE, Mode MODE>
int launch_side(const ProdArgs& p, bool a_kc, bool b_kc, hipStream_t s) {
  int rc;
  if constexpr (SIDE == kSide[kMid]) {
    if (!a_kc || !b_kc) return fail(MFX_E_INVALID, "no such product");
    rc = p.two ? launch<Cfg<SIDE, true, true, true>, MODE>(p, s) : launch<Cfg<SIDE, true, true, false>, MODE>(p, s);
  } else if (!a_kc) {
    // (Only a tall matrix's gram product reads columns of both.)
    if constexpr (MODE == kGram)
      rc = p.two ? launch<Cfg<SIDE, false, false, true>, MODE>(p, s) : launch<Cfg<SIDE, false, false, false>, MODE>(p, s);
    else
      return fail(MFX_E_INVALID, "no such product");
  } else if (!b_kc) {
    if constexpr (MODE == kApply)
      rc = p.two ? launch<Cfg<SIDE, true, false, true>, MODE>(p, s) : launch<Cfg<SIDE, true, false, false>, MODE>(p, s);
    else
      return fail(MFX_E_INVALID, "no such product");
  } else {
    rc = p.two ? launch<Cfg<SIDE, true, true, true>, MODE>(p, s) : launch<Cfg<SIDE, true, true, false>, MODE>(p, s);
  }
  if (rc || !p.splits) return rc;
  typedef Cfg<SIDE, true, true, false> J;
  const int64_t blocks = (p.all - p.whole) * J::NW * J::FM * J::FN;
  hipLaunchKernelGGL((ns_join<J, MODE>), dim3((unsigned)(blocks / kJoinWaves)), dim3(kJoinWaves * 64), 0, s, p);
  return launch_status("ns_join");
}

template <Mode MODE>
int product(ProdArgs& p, const Way& way, int64_t B, int64_t M, int64_t N, int64_t K, bool a_kc, bool b_kc, float* part,
            hipStream_t s) {
  const int side = kSide[way.form];
  p.g.M = (int)M, p.g.N = (int)N, p.g.K = (int)K;
  p.g.tiles_m = (int)ceil_div(M, side), p.g.tiles_n = (int)ceil_div(N, side);
  p.symmetric = MODE != kApply;
  p.tiles = way.tiles / B, p.all = way.tiles, p.whole = way.whole;
  p.splits = way.splits, p.per = way.per;
  p.kt = (int)ceil_div(K, depth(way.form, p.two));
  p.part = part;
  if (way.form == kWide) return launch_side<256, MODE>(p, a_kc, b_kc, s);
  if (way.form == kNarrow) return launch_side<128, MODE>(p, a_kc, b_kc, s);
  if (way.form == kMid) return launch_side<192, MODE>(p, a_kc, b_kc, s);
  return launch_side<64, MODE>(p, a_kc, b_kc, s);
}

// Everything behind the checks.  in: g, buf and their strides; last: where the result goes.
int run(const Plan& pl, InArgs in, const float* coeffs, int num_coeffs, const ProdArgs& last, float scale, char* ws,
        hipStream_t s) {
  double* const norm = reinterpret_cast<double*>(ws);
  uint16_t* x[2];
  x[0] = reinterpret_cast<uint16_t*>(ws + pl.norm_bytes);
  x[1] = reinterpret_cast<uint16_t*>(ws + pl.norm_bytes + pl.x_bytes);
  uint16_t* const a = reinterpret_cast<uint16_t*>(ws + pl.norm_bytes + 2 * pl.x_bytes);
  uint16_t* const q = reinterpret_cast<uint16_t*>(ws + pl.norm_bytes + 2 * pl.x_bytes + pl.a_bytes);
  uint16_t* const t = reinterpret_cast<uint16_t*>(ws + pl.norm_bytes + 2 * pl.x_bytes + 2 * pl.a_bytes);
  float* const part = reinterpret_cast<float*>(ws + pl.total - pl.part);
  const int64_t xs = pl.m * pl.ld, as = pl.s * pl.lds;
  in.norm = norm;
  in.x = x[0];
  in.lo = pl.B * xs;
  in.m = (int)pl.m, in.n = (int)pl.n, in.ld = (int)pl.ld, in.parts = pl.parts, in.two = pl.two;
  in.scale = pl.ex[0];
  hipLaunchKernelGGL(ns_norm, dim3(pl.parts, (unsigned)pl.B), dim3(256), 0, s, in);
  if (int rc = launch_status("ns_norm")) return rc;
  const int64_t chunks = ceil_div(pl.m * (pl.ld / 8), 256);
  hipLaunchKernelGGL(ns_split, dim3((unsigned)std::min<int64_t>(chunks, 2048), (unsigned)pl.B), dim3(256), 0, s, in);
  if (int rc = launch_status("ns_split")) return rc;
  auto of = [&](uint16_t* p) { return Operand{p, pl.lds, pl.B * as}; };
  // to = factor left right, of matrices of the smaller side
  auto small = [&](uint16_t* to, uint16_t* left, uint16_t* right, float factor) {
    ProdArgs p{};
    p.two = pl.two;
    p.g.a = of(left), p.g.b = of(right);
    p.as = p.bs = as;
    p.c = to, p.ldc = pl.lds, p.cs = as, p.lo = pl.B * as;
    p.c1 = factor;
    return product<kGram>(p, pl.small, pl.B, pl.s, pl.s, pl.s, true, true, part, s);
  };
  // to = step i's Q of A
  auto square = [&](uint16_t* to, uint16_t* from, int i) {
    const float* k = coeffs + 3 * (num_coeffs == 1 ? 0 : i);
    const float ea = pl.ea[i], eq = pl.eq[i];
    ProdArgs p{};
    p.two = pl.two;
    p.g.a = p.g.b = of(from);
    p.as = p.bs = as;
    p.c = to, p.ldc = pl.lds, p.cs = as, p.lo = pl.B * as;
    p.c1 = k[2] * eq / (ea * ea);
    p.c2 = k[1] * eq / ea;
    p.c3 = k[0] * eq;
    return product<kSquare>(p, pl.square, pl.B, pl.s, pl.s, pl.s, true, true, part, s);
  };
  for (int i = 0, turn = 0; i < pl.steps; turn ^= 1) {
    const Operand X{x[turn], pl.ld, pl.B * xs};
    ProdArgs p{};
    p.two = pl.two;
    p.g.a = p.g.b = X;
    p.as = p.bs = xs;
    p.c = a, p.ldc = pl.lds, p.cs = as, p.lo = pl.B * as;
    p.c1 = pl.ea[i] / (pl.ex[i] * pl.ex[i]);
    if (int rc = product<kGram>(p, pl.gram, pl.B, pl.s, pl.s, pl.l, pl.wide, pl.wide, part, s)) return rc;
    if (int rc = square(q, a, i)) return rc;
    const float ex = pl.ex[i];
    float by = pl.eq[i];  // what the factor of X is stored at, and where it is
    uint16_t* f = q;
    if (pl.paired && i + 1 < pl.steps) {
      const float eq = pl.eq[i], et = pl.et[i];
      if (int rc = small(t, q, a, et / (eq * pl.ea[i]))) return rc;
      if (int rc = small(a, t, q, pl.ea[i + 1] / (et * eq))) return rc;
      if (int rc = square(t, a, i + 1)) return rc;
      by = pl.ep[i];
      f = a;
      if (int rc = small(a, t, q, by / (pl.eq[i + 1] * eq))) return rc;
      ++i;
    }
    if (++i == pl.steps) {
      p = last;
      p.two = pl.two;
      p.c1 = scale / (by * ex);
    } else {
      p.c = x[turn ^ 1], p.ldc = pl.ld, p.cs = xs, p.lo = pl.B * xs;
      p.c1 = pl.ex[i] / (by * ex);
    }
    // Wide: Q's rows by X's columns; tall: X's rows by Q's (Q is symmetric).
    const Operand Q = of(f);
    p.g.a = pl.wide ? Q : X, p.as = pl.wide ? as : xs;
    p.g.b = pl.wide ? X : Q, p.bs = pl.wide ? xs : as;
    if (int rc = product<kApply>(p, pl.apply, pl.B, pl.m, pl.n, pl.s, true, !pl.wide, part, s)) return rc;
  }
  return MFX_OK;
}

int bind(const void* p, int64_t row, int64_t batch, const Plan& pl, int dt, const char* what, bool written) {
  if (!float_dtype(dt)) return fail(MFX_E_UNSUPPORTED, std::string(what) + ": dtype must be f32, bf16 or f16");
  if (pl.B == 0) return MFX_OK;
  if (!p) return fail(MFX_E_INVALID, std::string(what) + " must be non-null");
  if ((uintptr_t)p % dtype_size(dt)) return fail(MFX_E_INVALID, std::string(what) + " must be aligned to its type");
  if (pl.m > 1 && row < (written ? pl.n : 0)) return fail(MFX_E_INVALID, std::string(what) + ": row stride too small");
  if (pl.B > 1 && (batch < 0 || (written && batch < (pl.m - 1) * row + pl.n)))
    return fail(MFX_E_INVALID, std::string(what) + ": matrices must not overlap");
  return MFX_OK;
}

int plan_ns(const mfx_newton_schulz_args* a, Plan& pl) {
  if (!a) return fail(MFX_E_INVALID, "null args");
  if (int rc = plan_common(pl, a->batch, a->m, a->n, a->steps, a->coeffs, a->num_coeffs, a->eps, a->terms))
    return rc;
  if (!std::isfinite(a->scale)) return fail(MFX_E_INVALID, "scale must be finite");
  if (int rc = bind(a->g, a->g_row_stride, a->g_batch_stride, pl, a->dtype, "g", false)) return rc;
  return bind(a->out, a->out_row_stride, a->out_batch_stride, pl, a->out_dtype, "out", true);
}

int plan_muon(const mfx_muon_update_args* a, Plan& pl) {
  if (!a) return fail(MFX_E_INVALID, "null args");
  if (int rc = plan_common(pl, a->batch, a->m, a->n, a->steps, a->coeffs, a->num_coeffs, a->eps, a->terms))
    return rc;
  if (!std::isfinite(a->lr) || !std::isfinite(a->scale) || !std::isfinite(a->weight_decay))
    return fail(MFX_E_INVALID, "lr, scale and weight_decay must be finite");
  if (!(a->mu >= 0.f && a->mu <= 1.f)) return fail(MFX_E_INVALID, "mu must be within [0, 1]");
  if (int rc = bind(a->g, a->g_row_stride, a->g_batch_stride, pl, a->dtype, "g", false)) return rc;
  if (int rc = bind(a->w, a->w_row_stride, a->w_batch_stride, pl, a->w_dtype, "w", false)) return rc;
  if (int rc = bind(a->w_out, a->w_out_row_stride, a->w_out_batch_stride, pl, a->w_dtype, "w_out", true)) return rc;
  if ((a->momentum == nullptr) != (a->momentum_out == nullptr))
    return fail(MFX_E_INVALID, "momentum and momentum_out go together");
  if (!a->momentum) return MFX_OK;
  if (int rc = bind(a->momentum, a->momentum_row_stride, a->momentum_batch_stride, pl, a->momentum_dtype, "momentum", false))
    return rc;
  return bind(a->momentum_out, a->momentum_out_row_stride, a->momentum_out_batch_stride, pl, a->momentum_dtype,
              "momentum_out", true);
}

}  // namespace
}  // namespace ns
}  // namespace mfx

extern "C" {

size_t mfx_newton_schulz_workspace_size(const mfx_newton_schulz_args* args) {
  mfx::ns::Plan pl{};
  return mfx::ns::plan_ns(args, pl) == MFX_OK ? pl.total : 0;
}

int mfx_newton_schulz(const mfx_newton_schulz_args* args, void* stream) {
  using namespace mfx;
  using namespace mfx::ns;
  Plan pl{};
  if (int rc = plan_ns(args, pl)) return rc;
  const mfx_newton_schulz_args& a = *args;
  if (a.batch == 0) return MFX_OK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* ws = nullptr;
  if (int rc = take_workspace(a.workspace, a.workspace_bytes, pl.total, "mfx_newton_schulz_workspace_size", s, &ws))
    return rc;
  InArgs in{};
  in.g = a.g, in.gs_b = a.g_batch_stride, in.gs_r = a.g_row_stride, in.g_dt = a.dtype;
  in.eps = a.eps;
  ProdArgs last{};
  last.out = a.out, last.out_dt = a.out_dtype, last.os_b = a.out_batch_stride, last.os_r = a.out_row_stride;
  return run(pl, in, a.coeffs, a.num_coeffs, last, a.scale, ws, s);
}

size_t mfx_muon_update_workspace_size(const mfx_muon_update_args* args) {
  mfx::ns::Plan pl{};
  return mfx::ns::plan_muon(args, pl) == MFX_OK ? pl.total : 0;
}

int mfx_muon_update(const mfx_muon_update_args* args, void* stream) {
  using namespace mfx;
  using namespace mfx::ns;
  Plan pl{};
  if (int rc = plan_muon(args, pl)) return rc;
  const mfx_muon_update_args& a = *args;
  if (a.batch == 0) return MFX_OK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* ws = nullptr;
  if (int rc = take_workspace(a.workspace, a.workspace_bytes, pl.total, "mfx_muon_update_workspace_size", s, &ws))
    return rc;
  InArgs in{};
  in.g = a.g, in.gs_b = a.g_batch_stride, in.gs_r = a.g_row_stride, in.g_dt = a.dtype;
  in.buf = a.momentum, in.bs_b = a.momentum_batch_stride, in.bs_r = a.momentum_row_stride, in.buf_dt = a.momentum_dtype;
  in.buf_out = a.momentum_out, in.os_b = a.momentum_out_batch_stride, in.os_r = a.momentum_out_row_stride;
  in.eps = a.eps, in.mu = a.mu, in.nesterov = a.nesterov != 0;
  ProdArgs last{};
  last.out = a.w_out, last.out_dt = a.w_dtype, last.os_b = a.w_out_batch_stride, last.os_r = a.w_out_row_stride;
  last.w = a.w, last.ws_b = a.w_batch_stride, last.ws_r = a.w_row_stride;
  last.keep = 1.f - a.lr * a.weight_decay;
  return run(pl, in, a.coeffs, a.num_coeffs, last, -a.lr * a.scale, ws, s);
}

}  // extern "C"

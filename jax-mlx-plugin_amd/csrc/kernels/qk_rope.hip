// RMSNorm of each query and key head with the rotation by the token's
// position, and the backward of the pair.  Per head row x of D features,
// weight w, position(s) p of the token:
//
//   y = x * r * w,  r = 1 / sqrt(mean(x^2) + eps)
//   pair i of the first `rot` features (a, b) -> (a c_i - b s_i, b c_i + a s_i),
//   c_i, s_i = cos, sin of p_axis(i) * f_i;  features from rot on pass.
//
// and backward, for the gradient g of the output: u = R^T g (the rotation by
// the negative angle), dw = sum over rows of u x r,
// dx = r * (u w - x r * mean(u w x r)).
//
// Angles.  A frequency is held as a 64-bit fraction of a turn per position
// (F = f / 2 pi * 2^64, modulo whole turns), so position * F modulo 2^64 is
// the angle's fraction of a turn, exact but for F's own rounding: off by at
// most |p| * 2^-65 turns, 2^-34 for any 32-bit position, where the fp32
// product p * f of a far position has lost the angle altogether.  The top 32
// bits give a quadrant and a remainder within pi/4 of it, and sine and cosine
// of that are their Taylor polynomials (to x^9 and x^10: truncated by less
// than 2e-9 there).
//
// Layout.  A lane owns 2 VEC features of a row (two chunks of VEC: for pairs
// half the rotated features apart the chunks hold the two members, for pairs
// side by side they are neighbours), a row takes the power of two of lanes
// that covers it (8 at D = 128 in 16 bits), and a wavefront owns a token and
// walks the heads of its queries or of its keys (so one weight, and in the
// backward one set of sums, is all a lane holds).  The token's angles are
// formed once, a pair a lane, and handed round through LDS.  The next rows are
// on their way while these are worked on, as they came (unpacked when their
// turn comes: twice the registers would halve the wavefronts in flight).  A call
// of few tokens splits the heads over more wavefronts.  Everything is fp32 and
// rounded once, at the store.
//
// What bounds it: HBM, each row read once and written once (backward: two
// rows read, one written).  8192 tokens of 32 + 8 heads of 128, bf16: forward
// 32 us (168 MB, 5.2 TB/s; a copy runs at 4.8), backward 47 us (253 MB, 5.4
// TB/s) and 4 us for the weights' sums.  64 tokens: 5 us, one pass of rows after
// the other (position, angles, row, store), which is why their heads are split.
// Angles formed by every lane for its own pairs, in place of once a token: 46
// and 103 us.  4099 tokens of 16 + 16 heads of 96, f16, pairs side by side and
// three axes: 16 us (51 MB, 3.2 TB/s).  There a lane's two chunks are neighbours,
// so a load takes 16 of every 32 bytes, two lanes of a row's eight have no
// features, and two passes of rows stand behind each token's position and angles.
#include <algorithm>
#include <cmath>

#include "common.h"

namespace mfx {
namespace {

constexpr int kBlock = 256;
constexpr int kWaves = kBlock / 64;
constexpr int kMaxAxes = 4;
constexpr int kMaxD = 256;
constexpr int kMaxPartials = 1024;  // workgroups of the backward, and rows of its partial sums

struct Rows {  // one [B, H, T, D] tensor: strides (batch, head, seq) in elements
  const void* p;
  int64_t s[3];
};

struct Side {  // the queries', or the keys', part of a call
  Rows in, grad, out;  // (grad: of the outputs; out: dq or dk in the backward)
  const void* w;
  int heads, per_wave, parts;  // heads a wavefront walks, and wavefronts for all
};

struct Params {
  Side side[2];
  const int32_t* pos;
  const uint64_t* freqs;
  float* partial;  // [workgroups][D], the queries' first, or null
  int64_t ps[3];   // positions: strides (axis, batch, seq)
  uint32_t tokens;  // B * T, below 2^31
  uint32_t T;
  int D, rot, pairs;  // pairs = rot / 2
  int bound[kMaxAxes];  // pair i belongs to the first axis with i < bound
  float eps;
};

template <typename T, int VEC>
struct Chunk {
  typedef T type __attribute__((ext_vector_type(VEC)));
};
template <typename T>
struct Chunk<T, 1> {
  typedef T type;
};

template <typename T, int VEC>
__device__ __forceinline__ void unpack(const typename Chunk<T, VEC>::type& c, float* v) {
  if constexpr (VEC == 1) v[0] = to_f32(c);
  else
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = to_f32(static_cast<T>(c[j]));
}

template <typename T, int VEC>
__device__ __forceinline__ void store_chunk(T* p, const float* v) {
  typename Chunk<T, VEC>::type c;
  if constexpr (VEC == 1) c = from_f32<T>(v[0]);
  else
#pragma unroll
    for (int j = 0; j < VEC; ++j) c[j] = from_f32<T>(v[j]);
  *reinterpret_cast<typename Chunk<T, VEC>::type*>(p) = c;
}

// cos and sin of `turns` / 2^64 turns.
__device__ __forceinline__ void cos_sin(uint64_t turns, float& c, float& s) {
  const int32_t t = (int32_t)(turns >> 32);
  const uint32_t quarter = ((uint32_t)t + 0x20000000u) >> 30;
  const int32_t rem = (int32_t)((uint32_t)t - (quarter << 30));  // within 2^29: an eighth of a turn
  const float x = (float)rem * 1.46291807926715968e-9f;          // 2 pi / 2^32
  const float z = x * x;
  float sn = fmaf(z, 1.f / 362880.f, -1.f / 5040.f);
  sn = fmaf(z, sn, 1.f / 120.f);
  sn = fmaf(z, sn, -1.f / 6.f);
  sn = fmaf(x * z, sn, x);
  float cs = fmaf(z, -1.f / 3628800.f, 1.f / 40320.f);
  cs = fmaf(z, cs, -1.f / 720.f);
  cs = fmaf(z, cs, 1.f / 24.f);
  cs = fmaf(z, cs, -0.5f);
  cs = fmaf(z, cs, 1.f);
  const float a = (quarter & 1) ? sn : cs, b = (quarter & 1) ? cs : sn;
  c = (quarter == 1 || quarter == 2) ? -a : a;
  s = (quarter & 2) ? -b : b;
}

// A row's chunks of one lane, as they are in memory.
template <typename T, int VEC, int NU>
struct Raw {
  typename Chunk<T, VEC>::type c[NU][2];
  __device__ __forceinline__ void get(float (&v)[NU][2 * VEC]) const {
#pragma unroll
    for (int n = 0; n < NU; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) unpack<T, VEC>(c[n][h], &v[n][h * VEC]);
  }
};

// What a lane owns of every row: NU units of 2 VEC features.  Unit u < units
// of rotated pairs holds pairs u*VEC .. u*VEC + VEC-1; the units after them
// the features from rot on.
template <int VEC, int NU, int LPR, bool IL>
struct Unit {
  int off[NU][2];  // first feature of each chunk; -1: none
  bool turn[NU];   // rotated
  float c[NU][VEC], s[NU][VEC];
  __device__ __forceinline__ Unit(const Params& p, int l) {
    const int rotated = p.pairs / VEC;
#pragma unroll
    for (int n = 0; n < NU; ++n) {
      const int u = n * LPR + l;
      turn[n] = u < rotated;
      if (turn[n]) {
        off[n][0] = IL ? u * 2 * VEC : u * VEC;
        off[n][1] = IL ? u * 2 * VEC + VEC : p.pairs + u * VEC;
      } else {
        const int f = p.rot + (u - rotated) * 2 * VEC;
        off[n][0] = f < p.D ? f : -1;
        off[n][1] = f + VEC < p.D ? f + VEC : -1;
      }
    }
  }
  // cos and sin of token (b, t): pair lane, lane + 64, .. by each lane into the
  // wavefront's `cs`, from where every lane takes those of its own pairs.
  __device__ __forceinline__ void angles(const Params& p, int lane, int l, uint32_t b, uint32_t t,
                                         float (&cs)[2][kMaxD / 2]) {
    const int32_t* at = p.pos + b * p.ps[1] + t * p.ps[2];
    __builtin_amdgcn_wave_barrier();
    for (int i = lane; i < p.pairs; i += 64) {
      const int axis = (i >= p.bound[0]) + (i >= p.bound[1]) + (i >= p.bound[2]);
      const int64_t pos = at[axis * p.ps[0]];
      cos_sin((uint64_t)pos * p.freqs[i], cs[0][i], cs[1][i]);
    }
    // (One wavefront: its LDS operations are in order.)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int n = 0; n < NU; ++n) {
      const int i0 = turn[n] ? (n * LPR + l) * VEC : 0;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        c[n][j] = cs[0][i0 + j];
        s[n][j] = cs[1][i0 + j];
      }
    }
  }
  // Rotates (forward) or turns back (!FWD) the unit's 2 VEC values.
  template <bool FWD>
  __device__ __forceinline__ void rotate(int n, float* v) const {
    if (!turn[n]) return;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int ia = IL ? 2 * j : j, ib = IL ? 2 * j + 1 : VEC + j;
      const float a = v[ia], b = v[ib], sj = FWD ? s[n][j] : -s[n][j];
      v[ia] = a * c[n][j] - b * sj;
      v[ib] = b * c[n][j] + a * sj;
    }
  }
  template <typename T>
  __device__ __forceinline__ void load(const T* row, bool valid, Raw<T, VEC, NU>& r) const {
#pragma unroll
    for (int n = 0; n < NU; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        r.c[n][h] = typename Chunk<T, VEC>::type{};
        if (valid && off[n][h] >= 0)
          r.c[n][h] = *reinterpret_cast<const typename Chunk<T, VEC>::type*>(row + off[n][h]);
      }
  }
  template <typename T>
  __device__ __forceinline__ void store(T* row, const float (&v)[NU][2 * VEC]) const {
#pragma unroll
    for (int n = 0; n < NU; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (off[n][h] >= 0) store_chunk<T, VEC>(row + off[n][h], &v[n][h * VEC]);
  }
  template <typename PT>
  __device__ __forceinline__ void weight(const void* w, float (&v)[NU][2 * VEC]) const {
#pragma unroll
    for (int n = 0; n < NU; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          v[n][h * VEC + j] = w && off[n][h] >= 0 ? to_f32(static_cast<const PT*>(w)[off[n][h] + j]) : 1.f;
  }
};

template <typename T>
__device__ __forceinline__ T* row_of(const Rows& r, uint32_t b, int h, uint32_t t) {
  return const_cast<T*>(static_cast<const T*>(r.p)) + b * r.s[0] + h * r.s[1] + t * r.s[2];
}

// This workgroup's side and heads [h0, h1): blockIdx.y counts the queries'
// parts, then the keys'.
__device__ __forceinline__ const Side& my_side(const Params& p, int& h0, int& h1) {
  const bool key = (int)blockIdx.y >= p.side[0].parts;
  const Side& sd = p.side[key];
  h0 = ((int)blockIdx.y - (key ? p.side[0].parts : 0)) * sd.per_wave;
  h1 = min(sd.heads, h0 + sd.per_wave);
  return sd;
}

template <typename T, typename PT, int VEC, int NU, int LPR, bool IL>
__global__ __launch_bounds__(kBlock) void qk_rope_kernel(Params p) {
  constexpr int RPW = 64 / LPR;  // rows a wavefront holds at once
  __shared__ __attribute__((aligned(16))) float cs[kWaves][2][kMaxD / 2];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l = lane % LPR, g = lane / LPR;
  const uint32_t tok = blockIdx.x * kWaves + wave;
  if (tok >= p.tokens) return;
  const uint32_t b = tok / p.T, t = tok - b * p.T;
  int h0, h1;
  const Side& sd = my_side(p, h0, h1);

  Unit<VEC, NU, LPR, IL> u(p, l);
  Raw<T, VEC, NU> raw;
  u.load(row_of<T>(sd.in, b, min(h0 + g, h1 - 1), t), h0 + g < h1, raw);
  float w[NU][2 * VEC];
  u.template weight<PT>(sd.w, w);
  u.angles(p, lane, l, b, t, cs[wave]);
  const float inv_d = 1.f / (float)p.D;
  for (int h = h0 + g; h < h1 + g; h += RPW) {
    float x[NU][2 * VEC];
    raw.get(x);
    if (h - g + RPW < h1) u.load(row_of<T>(sd.in, b, min(h + RPW, h1 - 1), t), h + RPW < h1, raw);
    if (p.eps >= 0.f) {
      float ss = 0.f;
#pragma unroll
      for (int n = 0; n < NU; ++n)
#pragma unroll
        for (int j = 0; j < 2 * VEC; ++j) ss = fmaf(x[n][j], x[n][j], ss);
      const float r = 1.f / sqrtf(group_sum<LPR>(ss) * inv_d + p.eps);
#pragma unroll
      for (int n = 0; n < NU; ++n)
#pragma unroll
        for (int j = 0; j < 2 * VEC; ++j) x[n][j] = x[n][j] * r * w[n][j];
    }
#pragma unroll
    for (int n = 0; n < NU; ++n) u.template rotate<true>(n, x[n]);
    if (h < h1) u.store(row_of<T>(sd.out, b, h, t), x);
  }
}

// Backward.  A workgroup walks tokens in strides of the grid, each wavefront
// one token at a time; its lanes keep running weight gradients of the features
// they own, folded at the end into the workgroup's row of partial sums (in
// LDS, group after group in a fixed order), which qk_rope_params adds up.
template <typename T, typename PT, int VEC, int NU, int LPR, bool IL>
__global__ __launch_bounds__(kBlock) void qk_rope_bwd_kernel(Params p) {
  constexpr int RPW = 64 / LPR;
  __shared__ __attribute__((aligned(16))) float cs[kWaves][2][kMaxD / 2];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l = lane % LPR, g = lane / LPR;
  int h0, h1;
  const Side& sd = my_side(p, h0, h1);
  Unit<VEC, NU, LPR, IL> u(p, l);
  float w[NU][2 * VEC], acc[NU][2 * VEC];
  u.template weight<PT>(sd.w, w);
#pragma unroll
  for (int n = 0; n < NU; ++n)
#pragma unroll
    for (int j = 0; j < 2 * VEC; ++j) acc[n][j] = 0.f;
  const float inv_d = 1.f / (float)p.D;

  // Rows of (token, heads from h on) travel while the ones before are worked
  // on, across tokens too.
  Raw<T, VEC, NU> rx, rd;
  auto fetch = [&](uint32_t tok, int h) __attribute__((always_inline)) {
    const uint32_t b = tok / p.T, t = tok - b * p.T;
    const bool valid = h + g < h1;
    const int hh = valid ? h + g : h0;
    u.load(row_of<T>(sd.in, b, hh, t), valid, rx);
    u.load(row_of<T>(sd.grad, b, hh, t), valid, rd);
  };
  const uint32_t stride = gridDim.x * kWaves;
  uint32_t tok = blockIdx.x * kWaves + wave;
  if (tok < p.tokens) fetch(tok, h0);
  for (int hb = h0; tok < p.tokens;) {
    const uint32_t b = tok / p.T, t = tok - b * p.T;
    if (hb == h0) u.angles(p, lane, l, b, t, cs[wave]);
    const bool same = hb + RPW < h1;
    const uint32_t tok2 = same ? tok : tok + stride;
    const int hb2 = same ? hb + RPW : h0;
    float x[NU][2 * VEC], d[NU][2 * VEC];
    rx.get(x);
    rd.get(d);
    if (tok2 < p.tokens) fetch(tok2, hb2);
    const bool valid = hb + g < h1;
#pragma unroll
    for (int n = 0; n < NU; ++n) u.template rotate<false>(n, d[n]);
    if (p.eps >= 0.f) {
      float ss = 0.f;
#pragma unroll
      for (int n = 0; n < NU; ++n)
#pragma unroll
        for (int j = 0; j < 2 * VEC; ++j) ss = fmaf(x[n][j], x[n][j], ss);
      const float mean = group_sum<LPR>(ss) * inv_d;
      // (An absent row adds nothing: with eps = 0 its r would be infinite.)
      const float r = valid ? 1.f / sqrtf(mean + p.eps) : 0.f;
      float dot = 0.f;
#pragma unroll
      for (int n = 0; n < NU; ++n)
#pragma unroll
        for (int j = 0; j < 2 * VEC; ++j) {
          x[n][j] *= r;
          acc[n][j] = fmaf(d[n][j], x[n][j], acc[n][j]);
          d[n][j] *= w[n][j];
          dot = fmaf(d[n][j], x[n][j], dot);
        }
      const float m = group_sum<LPR>(dot) * inv_d;
#pragma unroll
      for (int n = 0; n < NU; ++n)
#pragma unroll
        for (int j = 0; j < 2 * VEC; ++j) d[n][j] = r * (d[n][j] - x[n][j] * m);
    }
    if (valid) u.store(row_of<T>(sd.out, b, hb + g, t), d);
    tok = tok2;
    hb = hb2;
  }
  if (!p.partial) return;  // (uniform over the grid)
  // Fold the rows a wavefront holds, then the wavefronts.
  __shared__ float fold[kWaves][kMaxD];
#pragma unroll
  for (int n = 0; n < NU; ++n)
#pragma unroll
    for (int j = 0; j < 2 * VEC; ++j) {
#pragma unroll
      for (int off = LPR; off < 64; off <<= 1) acc[n][j] += __shfl_xor(acc[n][j], off, 64);
      const int h = j / VEC;
      if (g == 0 && u.off[n][h] >= 0) fold[wave][u.off[n][h] + j % VEC] = acc[n][j];
    }
  __syncthreads();
  float* out = p.partial + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * p.D;
  for (int i = threadIdx.x; i < p.D; i += kBlock) {
    float s = 0.f;
#pragma unroll
    for (int wv = 0; wv < kWaves; ++wv) s += fold[wv][i];
    out[i] = s;
  }
}

// dw[d] = sum over the G0 partial rows of the queries (blockIdx.y 0) or the G1
// behind them of the keys, 16 columns a workgroup, each column's rows shared
// out over 64 threads (eight in flight at a time) and folded in order.
template <typename PT>
__global__ __launch_bounds__(1024) void qk_rope_params(const float* __restrict__ partial, int G0, int G1, int D,
                                                       PT* dqw, PT* dkw) {
  PT* const out = blockIdx.y ? dkw : dqw;
  if (!out) return;
  const int G = blockIdx.y ? G1 : G0;
  if (blockIdx.y) partial += (int64_t)G0 * D;
  __shared__ float fold[64][17];
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
  const int col = blockIdx.x * 16 + c;
  float s = 0.f;
  if (col < D)
    for (int i0 = r; i0 < G; i0 += 8 * 64) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = i0 + u * 64 < G ? partial[(int64_t)(i0 + u * 64) * D + col] : 0.f;
#pragma unroll
      for (int u = 0; u < 8; ++u) s += v[u];
    }
  fold[r][c] = s;
  __syncthreads();
  if (r != 0 || col >= D) return;
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < 64; ++i) t += fold[i][c];
  out[col] = from_f32<PT>(t);
}

// ---- host ------------------------------------------------------------------

int pow2_at_least(int n) {
  int r = 1;
  while (r < n) r *= 2;
  return r;
}

struct Plan {
  Params p{};
  int vec = 1, nu = 1, lpr = 1;
  bool f32_params = true;
  dim3 grid;       // workgroups
  bool sums = false;  // the backward adds up weight gradients
};

bool float_dtype(int dt) { return dt == MFX_F32 || dt == MFX_BF16 || dt == MFX_F16; }

// One tensor's place in a plan: strides (batch, head, seq, feature).
int bind(Rows& r, const void* ptr, const int64_t* st, const char* what) {
  if (st[3] != 1) return fail(MFX_E_INVALID, std::string(what) + ": feature (last) stride must be 1");
  r.p = ptr;
  for (int i = 0; i < 3; ++i) r.s[i] = st[i];
  return MFX_OK;
}

bool chunked(const Rows& r, int vec, int size) {
  if (!r.p) return true;
  if ((uintptr_t)r.p % (uintptr_t)(vec * size)) return false;
  for (int i = 0; i < 3; ++i)
    if (r.s[i] % vec) return false;
  return true;
}

// Shared by both directions; the rows of `p` are bound already.
int plan_common(Plan& pl, int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t rot, const int32_t* pos,
                const uint64_t* freqs, const int64_t* ps, const int32_t* sections, int axes, float eps, int dtype,
                int param_dtype, bool il, bool weights) {
  Params& p = pl.p;
  const int64_t lim = 0x7fffffffLL;
  if (B < 0 || T < 0 || Hq < 0 || Hkv < 0 || Hq + Hkv <= 0 || D <= 0)
    return fail(MFX_E_INVALID, "B, T, Hq and Hkv must be >= 0, Hq + Hkv and D positive");
  if (D > kMaxD) return fail(MFX_E_UNSUPPORTED, "head size above 256 is not supported");
  if (B > lim || T > lim || Hq > 65535 || Hkv > 65535 || (T > 0 && B > lim / T))
    return fail(MFX_E_UNSUPPORTED, "problem too large for one launch");
  if (!float_dtype(dtype)) return fail(MFX_E_UNSUPPORTED, "dtype must be f32, bf16 or f16");
  if (weights && param_dtype != dtype && param_dtype != MFX_F32)
    return fail(MFX_E_UNSUPPORTED, "param_dtype must be dtype or f32");
  if (std::isnan(eps) || std::isinf(eps)) return fail(MFX_E_INVALID, "eps must be finite (negative: no norm)");
  if (eps < 0.f && weights) return fail(MFX_E_INVALID, "weights need a norm (eps >= 0)");
  if (rot < 0 || rot > D || rot % 2) return fail(MFX_E_INVALID, "rot must be even and within [0, D]");
  if (axes < 1 || axes > kMaxAxes) return fail(MFX_E_INVALID, "axes must be 1 to 4");
  if (rot > 0 && B * T > 0 && (!pos || !freqs)) return fail(MFX_E_INVALID, "a rotation needs positions and freqs");
  int64_t sum = 0;
  for (int a = 0; a < kMaxAxes; ++a) {
    if (a < axes) {
      if (sections[a] < 0) return fail(MFX_E_INVALID, "sections must be >= 0");
      sum += sections[a];
    }
    p.bound[a] = a < axes - 1 ? (int)sum : 0x7fffffff;
  }
  if (sum != rot / 2) return fail(MFX_E_INVALID, "sections must add up to rot / 2");
  p.pos = pos;
  p.freqs = freqs;
  for (int i = 0; i < 3; ++i) p.ps[i] = ps[i];
  p.tokens = (uint32_t)(B * T);
  p.T = (uint32_t)T;
  p.side[0].heads = (int)Hq;
  p.side[1].heads = (int)Hkv;
  p.D = (int)D;
  p.rot = (int)rot;
  p.pairs = (int)(rot / 2);
  p.eps = eps;
  pl.f32_params = !weights || param_dtype == MFX_F32;
  // The widest chunk that every row, the pairs and the rest divide into: 16
  // bytes, 8 bytes for 16-bit types, or single elements.
  const int size = dtype_size(dtype);
  const int widths[3] = {16 / size, 4, 1};
  for (int vec : widths) {
    if (D % vec || p.pairs % vec || (D - rot) % vec) continue;
    bool ok = true;
    for (const Side& sd : p.side)
      for (const Rows* r : {&sd.in, &sd.grad, &sd.out}) ok = ok && chunked(*r, vec, size);
    if (!ok) continue;
    pl.vec = vec;
    break;
  }
  const int units = p.pairs / pl.vec + (int)((D - rot + 2 * pl.vec - 1) / (2 * pl.vec));
  pl.nu = units > 64 ? 2 : 1;
  pl.lpr = pow2_at_least((units + pl.nu - 1) / pl.nu);
  if (pl.lpr < 4) pl.lpr = 4;
  return MFX_OK;
}

// Wavefronts that the tokens should be shared out to: eight a CU.
int64_t wanted_waves() { return 8LL * device_cu_count(); }

// Heads a wavefront walks: all of a side (its angles then serve them all) unless
// `waves` of them are fewer than wanted, when the heads are split down to one
// pass of rows each.
void split_heads(Plan& pl, int64_t waves) {
  const int rpw = 64 / pl.lpr;
  for (Side& sd : pl.p.side) {
    sd.parts = sd.per_wave = 0;
    if (sd.heads == 0) continue;
    const int passes = (sd.heads + rpw - 1) / rpw;
    const int64_t want = wanted_waves();
    const int parts = waves > 0 && waves < want ? (int)std::min<int64_t>(passes, (want + waves - 1) / waves) : 1;
    const int per = (passes + parts - 1) / parts;
    sd.per_wave = per * rpw;
    sd.parts = (passes + per - 1) / per;
  }
}

template <bool BWD, typename T, typename PT, int VEC, int NU, int LPR, bool IL>
void launch(const Plan& pl, hipStream_t s) {
  if constexpr (BWD)
    hipLaunchKernelGGL((qk_rope_bwd_kernel<T, PT, VEC, NU, LPR, IL>), pl.grid, dim3(kBlock), 0, s, pl.p);
  else hipLaunchKernelGGL((qk_rope_kernel<T, PT, VEC, NU, LPR, IL>), pl.grid, dim3(kBlock), 0, s, pl.p);
}

template <bool BWD, typename T, typename PT, int VEC, bool IL>
void launch_l(const Plan& pl, hipStream_t s) {
  if (pl.nu == 2) return launch<BWD, T, PT, VEC, VEC == 1 ? 2 : 1, 64, IL>(pl, s);
  switch (pl.lpr) {
    case 4: return launch<BWD, T, PT, VEC, 1, 4, IL>(pl, s);
    case 8: return launch<BWD, T, PT, VEC, 1, 8, IL>(pl, s);
    case 16: return launch<BWD, T, PT, VEC, 1, 16, IL>(pl, s);
    case 32: return launch<BWD, T, PT, VEC, 1, 32, IL>(pl, s);
    default: return launch<BWD, T, PT, VEC, 1, 64, IL>(pl, s);
  }
}

template <bool BWD, typename T, typename PT>
void launch_v(const Plan& pl, bool il, hipStream_t s) {
  constexpr int W = 16 / sizeof(T);
  if (pl.vec == W) return il ? launch_l<BWD, T, PT, W, true>(pl, s) : launch_l<BWD, T, PT, W, false>(pl, s);
  if constexpr (W != 4)
    if (pl.vec == 4) return il ? launch_l<BWD, T, PT, 4, true>(pl, s) : launch_l<BWD, T, PT, 4, false>(pl, s);
  return il ? launch_l<BWD, T, PT, 1, true>(pl, s) : launch_l<BWD, T, PT, 1, false>(pl, s);
}

template <bool BWD>
int launch_t(const Plan& pl, int dtype, bool il, hipStream_t s) {
  if (dtype == MFX_F32) launch_v<BWD, float, float>(pl, il, s);
  else if (dtype == MFX_BF16) {
    if (pl.f32_params) launch_v<BWD, bf16, float>(pl, il, s);
    else launch_v<BWD, bf16, bf16>(pl, il, s);
  } else {
    if (pl.f32_params) launch_v<BWD, _Float16, float>(pl, il, s);
    else launch_v<BWD, _Float16, _Float16>(pl, il, s);
  }
  return launch_status(BWD ? "qk_rope_bwd_kernel" : "qk_rope_kernel");
}

int plan_fwd(const mfx_qk_norm_rope_args* a, Plan& pl) {
  if (!a) return fail(MFX_E_INVALID, "null args");
  const bool any = a->B != 0 && a->T != 0;  // (an empty tensor may have no address)
  if (any && ((a->Hq > 0 && (!a->q || !a->q_out)) || (a->Hkv > 0 && (!a->k || !a->k_out))))
    return fail(MFX_E_INVALID, "q, q_out (and with Hkv > 0 k, k_out) must be non-null");
  Params& p = pl.p;
  Side &q = p.side[0], &k = p.side[1];
  int rc = MFX_OK;
  if (a->Hq > 0 && ((rc = bind(q.in, a->q, a->q_strides, "q")) || (rc = bind(q.out, a->q_out, a->qo_strides, "q_out"))))
    return rc;
  if (a->Hkv > 0 && ((rc = bind(k.in, a->k, a->k_strides, "k")) || (rc = bind(k.out, a->k_out, a->ko_strides, "k_out"))))
    return rc;
  q.w = a->q_weight;
  k.w = a->k_weight;
  rc = plan_common(pl, a->B, a->T, a->Hq, a->Hkv, a->D, a->rot, a->positions, a->freqs, a->pos_strides, a->sections,
                   a->axes, a->eps, a->dtype, a->param_dtype, a->interleaved != 0, a->q_weight || a->k_weight);
  if (rc) return rc;
  if (p.tokens == 0) return MFX_OK;
  const int64_t blocks = ((int64_t)p.tokens + kWaves - 1) / kWaves;
  if (!launch_fits(blocks, kBlock)) return fail(MFX_E_UNSUPPORTED, "problem too large for one launch");
  split_heads(pl, p.tokens);
  pl.grid = dim3((unsigned)blocks, (unsigned)(q.parts + k.parts));
  return MFX_OK;
}

int plan_bwd(const mfx_qk_norm_rope_bwd_args* a, Plan& pl) {
  if (!a) return fail(MFX_E_INVALID, "null args");
  const bool any = a->B != 0 && a->T != 0;
  if (any && ((a->Hq > 0 && (!a->q || !a->dq_out || !a->dq)) || (a->Hkv > 0 && (!a->k || !a->dk_out || !a->dk))))
    return fail(MFX_E_INVALID, "q, dq_out, dq (and with Hkv > 0 k, dk_out, dk) must be non-null");
  Params& p = pl.p;
  Side &q = p.side[0], &k = p.side[1];
  int rc = MFX_OK;
  if (a->Hq > 0 && ((rc = bind(q.in, a->q, a->q_strides, "q")) || (rc = bind(q.grad, a->dq_out, a->dqo_strides, "dq_out")) ||
                    (rc = bind(q.out, a->dq, a->dq_strides, "dq"))))
    return rc;
  if (a->Hkv > 0 && ((rc = bind(k.in, a->k, a->k_strides, "k")) ||
                     (rc = bind(k.grad, a->dk_out, a->dko_strides, "dk_out")) ||
                     (rc = bind(k.out, a->dk, a->dk_strides, "dk"))))
    return rc;
  q.w = a->q_weight;
  k.w = a->k_weight;
  const bool grads = a->dq_weight || a->dk_weight;
  rc = plan_common(pl, a->B, a->T, a->Hq, a->Hkv, a->D, a->rot, a->positions, a->freqs, a->pos_strides, a->sections,
                   a->axes, a->eps, a->dtype, a->param_dtype, a->interleaved != 0,
                   a->q_weight || a->k_weight || grads);
  if (rc) return rc;
  // Workgroups: one token a wavefront up to kMaxPartials of them, then each
  // wavefront walks several (fewer partial rows to add up).
  const int64_t blocks = std::min<int64_t>(((int64_t)p.tokens + kWaves - 1) / kWaves, kMaxPartials);
  split_heads(pl, blocks * kWaves);
  pl.grid = dim3((unsigned)blocks, (unsigned)(q.parts + k.parts));
  pl.sums = grads && p.tokens > 0;
  return MFX_OK;
}

size_t bwd_bytes(const Plan& pl) { return pl.sums ? (size_t)pl.grid.x * pl.grid.y * pl.p.D * sizeof(float) : 0; }

}  // namespace
}  // namespace mfx

extern "C" {

int mfx_rope_freqs(double theta, int64_t rot, const double* inv_freq, uint64_t* out) {
  using namespace mfx;
  if (!out || rot <= 0 || rot % 2) return fail(MFX_E_INVALID, "out must be non-null and rot positive and even");
  if (!inv_freq && !(theta > 0.0 && std::isfinite(theta)))
    return fail(MFX_E_INVALID, "theta must be positive and finite");
  const long double two_pi = 6.283185307179586476925286766559005768L;
  for (int64_t i = 0; i < rot / 2; ++i) {
    const long double f = inv_freq ? (long double)inv_freq[i] : powl((long double)theta, -2.0L * i / rot);
    if (!std::isfinite((double)f)) return fail(MFX_E_INVALID, "frequencies must be finite");
    long double turns = f / two_pi;
    turns -= floorl(turns);
    const long double scaled = rintl(ldexpl(turns, 64));
    // (A fraction that rounds to a whole turn is no turn at all.)
    out[i] = scaled >= 18446744073709551616.0L ? 0 : (uint64_t)scaled;
  }
  return MFX_OK;
}

int mfx_qk_norm_rope(const mfx_qk_norm_rope_args* args, void* stream) {
  using namespace mfx;
  Plan pl;
  if (int rc = plan_fwd(args, pl)) return rc;
  if (pl.p.tokens == 0) return MFX_OK;
  return launch_t<false>(pl, args->dtype, args->interleaved != 0, static_cast<hipStream_t>(stream));
}

size_t mfx_qk_norm_rope_bwd_workspace_size(const mfx_qk_norm_rope_bwd_args* args) {
  mfx::Plan pl;
  if (mfx::plan_bwd(args, pl) != MFX_OK) return 0;
  if (!pl.sums) return 0;
  // At any alignment: narrower chunks take more lanes a row, hence more parts
  // of the heads, up to one row each or what fills the device (split_heads).
  const int64_t waves = (int64_t)pl.grid.x * mfx::kWaves, want = mfx::wanted_waves();
  int64_t parts = 0;
  for (const mfx::Side& sd : pl.p.side)
    if (sd.heads) parts += waves < want ? std::min<int64_t>(sd.heads, (want + waves - 1) / waves) : 1;
  return (size_t)pl.grid.x * parts * pl.p.D * sizeof(float);
}

int mfx_qk_norm_rope_bwd(const mfx_qk_norm_rope_bwd_args* args, void* stream) {
  using namespace mfx;
  Plan pl;
  if (int rc = plan_bwd(args, pl)) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const size_t need = bwd_bytes(pl);
  if (need) {
    if (args->workspace) {
      if (args->workspace_bytes < need)
        return fail(MFX_E_WORKSPACE, "workspace smaller than mfx_qk_norm_rope_bwd_workspace_size()");
      if ((uintptr_t)args->workspace % 4) return fail(MFX_E_INVALID, "workspace must be 4-byte aligned");
      pl.p.partial = static_cast<float*>(args->workspace);
    } else {
      pl.p.partial = static_cast<float*>(device_scratch(need, s));
      if (!pl.p.partial) return MFX_E_HIP;
    }
  }
  if (pl.p.tokens > 0)
    if (int rc = launch_t<true>(pl, args->dtype, args->interleaved != 0, s)) return rc;
  if (!args->dq_weight && !args->dk_weight) return MFX_OK;
  // (Without tokens the weight gradients are empty sums.)
  const dim3 grid((unsigned)((pl.p.D + 15) / 16), 2);
  const int g0 = pl.sums ? (int)pl.grid.x * pl.p.side[0].parts : 0, g1 = pl.sums ? (int)pl.grid.x * pl.p.side[1].parts : 0;
  if (pl.f32_params)
    hipLaunchKernelGGL((qk_rope_params<float>), grid, dim3(1024), 0, s, pl.p.partial, g0, g1, pl.p.D,
                       static_cast<float*>(args->dq_weight), static_cast<float*>(args->dk_weight));
  else if (args->dtype == MFX_BF16)
    hipLaunchKernelGGL((qk_rope_params<bf16>), grid, dim3(1024), 0, s, pl.p.partial, g0, g1, pl.p.D,
                       static_cast<bf16*>(args->dq_weight), static_cast<bf16*>(args->dk_weight));
  else
    hipLaunchKernelGGL((qk_rope_params<_Float16>), grid, dim3(1024), 0, s, pl.p.partial, g0, g1, pl.p.D,
                       static_cast<_Float16*>(args->dq_weight), static_cast<_Float16*>(args->dk_weight));
  return launch_status("qk_rope_params");
}

}  // extern "C"

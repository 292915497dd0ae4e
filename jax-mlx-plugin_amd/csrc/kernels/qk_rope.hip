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
// walks its heads, queries first, so that a token's angles are formed once
// for all its heads.  A call of few tokens splits the heads over more
// wavefronts.  Everything is fp32 and rounded once, at the store.
//
// What bounds it: HBM, each row read once and written once (backward: two
// rows read, one written).
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

struct Params {
  Rows q, k;    // inputs
  Rows gq, gk;  // gradients of the outputs (backward)
  Rows qo, ko;  // outputs (backward: dq, dk)
  const void* qw;
  const void* kw;
  const int32_t* pos;
  const uint64_t* freqs;
  float* partial;  // [workgroups][2][D], or null
  int64_t ps[3];   // positions: strides (axis, batch, seq)
  int64_t tokens;  // B * T
  int64_t T;
  int Hq, H;       // query heads, all heads
  int D, rot, pairs;  // pairs = rot / 2
  int bound[kMaxAxes];  // pair i belongs to the first axis with i < bound
  int heads_per_wave;   // a multiple of the rows a wavefront holds at once
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
__device__ __forceinline__ void load_chunk(const T* p, float* v) {
  const auto c = *reinterpret_cast<const typename Chunk<T, VEC>::type*>(p);
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

// What a lane owns of every row: NU units of 2 VEC features.  Unit u < units
// of rotated pairs holds pairs u*VEC .. u*VEC + VEC-1; the units after them
// the features from rot on.
template <int VEC, int NU, int LPR, bool IL>
struct Unit {
  int off[NU][2];   // first feature of each chunk; -1: none
  bool turn[NU];    // rotated
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
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        c[n][j] = 1.f;
        s[n][j] = 0.f;
      }
    }
  }
  __device__ __forceinline__ void angles(const Params& p, int l, int64_t b, int64_t t) {
#pragma unroll
    for (int n = 0; n < NU; ++n) {
      if (!turn[n]) continue;
      const int i0 = (n * LPR + l) * VEC;
      const int32_t* at = p.pos + b * p.ps[1] + t * p.ps[2];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int i = i0 + j;
        const int axis = (i >= p.bound[0]) + (i >= p.bound[1]) + (i >= p.bound[2]);
        const int64_t pos = at[axis * p.ps[0]];
        cos_sin((uint64_t)pos * p.freqs[i], c[n][j], s[n][j]);
      }
    }
  }
  // Rotates (forward) or turns back (!FWD) the unit's 2 VEC values.
  template <bool FWD>
  __device__ __forceinline__ void rotate(int n, float* v) const {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int ia = IL ? 2 * j : j, ib = IL ? 2 * j + 1 : VEC + j;
      const float a = v[ia], b = v[ib], sj = FWD ? s[n][j] : -s[n][j];
      v[ia] = a * c[n][j] - b * sj;
      v[ib] = b * c[n][j] + a * sj;
    }
  }
  template <typename T>
  __device__ __forceinline__ void load(const T* row, bool valid, float (&v)[NU][2 * VEC]) const {
#pragma unroll
    for (int n = 0; n < NU; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (valid && off[n][h] >= 0) load_chunk<T, VEC>(row + off[n][h], &v[n][h * VEC]);
        else
#pragma unroll
          for (int j = 0; j < VEC; ++j) v[n][h * VEC + j] = 0.f;
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
};

template <typename PT, int VEC, int NU, class U>
__device__ __forceinline__ void load_weight(const U& u, const void* w, float (&v)[NU][2 * VEC]) {
#pragma unroll
  for (int n = 0; n < NU; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        v[n][h * VEC + j] = w && u.off[n][h] >= 0 ? to_f32(static_cast<const PT*>(w)[u.off[n][h] + j]) : 1.f;
}

// Row of head hh (queries first) of a (q, k) tensor pair.
template <typename T>
__device__ __forceinline__ const T* row_of(const Rows& q, const Rows& k, int Hq, int hh, int64_t b, int64_t t) {
  const bool isq = hh < Hq;
  const T* base = static_cast<const T*>(isq ? q.p : k.p);
  const int64_t* s = isq ? q.s : k.s;
  return base + b * s[0] + (int64_t)(isq ? hh : hh - Hq) * s[1] + t * s[2];
}

template <typename T, typename PT, int VEC, int NU, int LPR, bool IL>
__global__ __launch_bounds__(kBlock) void qk_rope_kernel(Params p) {
  constexpr int RPW = 64 / LPR;  // rows a wavefront holds at once
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l = lane % LPR, g = lane / LPR;
  const int64_t tok = (int64_t)blockIdx.x * kWaves + wave;
  if (tok >= p.tokens) return;
  const int64_t b = tok / p.T, t = tok % p.T;
  const int h0 = blockIdx.y * p.heads_per_wave;
  const int h1 = min(p.H, h0 + p.heads_per_wave);

  Unit<VEC, NU, LPR, IL> u(p, l);
  float x[NU][2 * VEC];
  int hh = h0 + g;
  if (hh < h1) u.load(row_of<T>(p.q, p.k, p.Hq, hh, b, t), true, x);
  u.angles(p, l, b, t);
  float qw[NU][2 * VEC], kw[NU][2 * VEC];
  load_weight<PT, VEC, NU>(u, p.qw, qw);
  load_weight<PT, VEC, NU>(u, p.kw, kw);
  const float inv_d = 1.f / (float)p.D;
  for (int hb = h0; hb < h1; hb += RPW, hh += RPW) {
    // The next head's row travels while this one is worked on.
    float nx[NU][2 * VEC];
    const bool more = hh + RPW < h1;
    u.load(row_of<T>(p.q, p.k, p.Hq, more ? hh + RPW : h0, b, t), more, nx);
    float ss = 0.f;
#pragma unroll
    for (int n = 0; n < NU; ++n)
#pragma unroll
      for (int j = 0; j < 2 * VEC; ++j) ss = fmaf(x[n][j], x[n][j], ss);
    const float r = p.eps >= 0.f ? 1.f / sqrtf(group_sum<LPR>(ss) * inv_d + p.eps) : 1.f;
    const bool isq = hh < p.Hq;
#pragma unroll
    for (int n = 0; n < NU; ++n) {
#pragma unroll
      for (int j = 0; j < 2 * VEC; ++j) x[n][j] = x[n][j] * r * (isq ? qw[n][j] : kw[n][j]);
      if (u.turn[n]) u.template rotate<true>(n, x[n]);
    }
    if (hh < h1) u.store(const_cast<T*>(row_of<T>(p.qo, p.ko, p.Hq, hh, b, t)), x);
#pragma unroll
    for (int n = 0; n < NU; ++n)
#pragma unroll
      for (int j = 0; j < 2 * VEC; ++j) x[n][j] = nx[n][j];
  }
}

// Backward.  A workgroup walks tokens in strides of the grid, each wavefront
// one token at a time; its lanes keep running weight gradients of the features
// they own, folded at the end into the workgroup's row of partial sums (in
// LDS, group after group in a fixed order), which qk_rope_params adds up.
template <typename T, typename PT, int VEC, int NU, int LPR, bool IL>
__global__ __launch_bounds__(kBlock) void qk_rope_bwd_kernel(Params p) {
  constexpr int RPW = 64 / LPR;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l = lane % LPR, g = lane / LPR;
  Unit<VEC, NU, LPR, IL> u(p, l);
  float qw[NU][2 * VEC], kw[NU][2 * VEC], aq[NU][2 * VEC], ak[NU][2 * VEC];
  load_weight<PT, VEC, NU>(u, p.qw, qw);
  load_weight<PT, VEC, NU>(u, p.kw, kw);
#pragma unroll
  for (int n = 0; n < NU; ++n)
#pragma unroll
    for (int j = 0; j < 2 * VEC; ++j) aq[n][j] = ak[n][j] = 0.f;
  const float inv_d = 1.f / (float)p.D;
  const int h0 = blockIdx.y * p.heads_per_wave;
  const int h1 = min(p.H, h0 + p.heads_per_wave);

  for (int64_t tok = (int64_t)blockIdx.x * kWaves + wave; tok < p.tokens; tok += (int64_t)gridDim.x * kWaves) {
    const int64_t b = tok / p.T, t = tok % p.T;
    u.angles(p, l, b, t);
    for (int hb = h0; hb < h1; hb += RPW) {
      const int hh = hb + g;
      const bool valid = hh < h1, isq = hh < p.Hq;
      float x[NU][2 * VEC], d[NU][2 * VEC];
      u.load(row_of<T>(p.q, p.k, p.Hq, valid ? hh : h0, b, t), valid, x);
      u.load(row_of<T>(p.gq, p.gk, p.Hq, valid ? hh : h0, b, t), valid, d);
      float ss = 0.f;
#pragma unroll
      for (int n = 0; n < NU; ++n) {
#pragma unroll
        for (int j = 0; j < 2 * VEC; ++j) ss = fmaf(x[n][j], x[n][j], ss);
        if (u.turn[n]) u.template rotate<false>(n, d[n]);
      }
      if (p.eps >= 0.f) {
        // (An absent row adds nothing: with eps = 0 its r would be infinite.)
        const float r = valid ? 1.f / sqrtf(group_sum<LPR>(ss) * inv_d + p.eps) : (group_sum<LPR>(ss), 0.f);
        float dot = 0.f;
#pragma unroll
        for (int n = 0; n < NU; ++n)
#pragma unroll
          for (int j = 0; j < 2 * VEC; ++j) {
            x[n][j] *= r;
            const float dxh = d[n][j] * x[n][j];
            if (isq) aq[n][j] += dxh;
            else ak[n][j] += dxh;
            d[n][j] *= isq ? qw[n][j] : kw[n][j];
            dot = fmaf(d[n][j], x[n][j], dot);
          }
        const float m = group_sum<LPR>(dot) * inv_d;
#pragma unroll
        for (int n = 0; n < NU; ++n)
#pragma unroll
          for (int j = 0; j < 2 * VEC; ++j) d[n][j] = r * (d[n][j] - x[n][j] * m);
      }
      if (valid) u.store(const_cast<T*>(row_of<T>(p.qo, p.ko, p.Hq, hh, b, t)), d);
    }
  }
  if (!p.partial) return;  // (uniform over the grid)
  // Fold the rows a wavefront holds, then the wavefronts.
  __shared__ float fold[kWaves][2][kMaxD];
#pragma unroll
  for (int n = 0; n < NU; ++n)
#pragma unroll
    for (int j = 0; j < 2 * VEC; ++j) {
#pragma unroll
      for (int off = LPR; off < 64; off <<= 1) {
        aq[n][j] += __shfl_xor(aq[n][j], off, 64);
        ak[n][j] += __shfl_xor(ak[n][j], off, 64);
      }
      const int h = j / VEC;
      if (g == 0 && u.off[n][h] >= 0) {
        fold[wave][0][u.off[n][h] + j % VEC] = aq[n][j];
        fold[wave][1][u.off[n][h] + j % VEC] = ak[n][j];
      }
    }
  __syncthreads();
  float* out = p.partial + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 * p.D;
  for (int i = threadIdx.x; i < 2 * p.D; i += kBlock) {
    const int which = i / p.D, d = i % p.D;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) s += fold[w][which][d];
    out[i] = s;
  }
}

// dw[which][d] = sum over the G partial rows, 32 columns a workgroup, each
// column's rows shared out over 32 threads and folded in order.
template <typename PT>
__global__ __launch_bounds__(1024) void qk_rope_params(const float* __restrict__ partial, int G, int D, PT* dqw,
                                                       PT* dkw) {
  __shared__ float fold[32][33];
  const int c = threadIdx.x & 31, r = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + c;
  float s = 0.f;
  if (col < 2 * D)
    for (int i = r; i < G; i += 32) s += partial[(int64_t)i * 2 * D + col];
  fold[r][c] = s;
  __syncthreads();
  if (r != 0 || col >= 2 * D) return;
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) t += fold[i][c];
  PT* out = col < D ? dqw : dkw;
  if (out) out[col < D ? col : col - D] = from_f32<PT>(t);
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
  int partials = 0;  // rows of partial sums (backward with weight gradients)
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
  p.tokens = B * T;
  p.T = T;
  p.Hq = (int)Hq;
  p.H = (int)(Hq + Hkv);
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
    for (const Rows* r : {&p.q, &p.k, &p.gq, &p.gk, &p.qo, &p.ko}) ok = ok && chunked(*r, vec, size);
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

// Heads a wavefront walks: all of them (its angles then serve the whole
// token) unless the tokens are too few to fill the device with eight
// wavefronts a CU, when they are split down to one pass of rows each.
// Returns the number of parts.
int split_heads(Plan& pl, int64_t waves) {
  const int rpw = 64 / pl.lpr;
  const int passes = (pl.p.H + rpw - 1) / rpw;
  const int64_t want = 8LL * device_cu_count();
  int parts = waves > 0 && waves < want ? (int)std::min<int64_t>(passes, (want + waves - 1) / waves) : 1;
  const int per = (passes + parts - 1) / parts;
  pl.p.heads_per_wave = per * rpw;
  return (passes + per - 1) / per;
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
  int rc = MFX_OK;
  if (a->Hq > 0 && ((rc = bind(p.q, a->q, a->q_strides, "q")) || (rc = bind(p.qo, a->q_out, a->qo_strides, "q_out"))))
    return rc;
  if (a->Hkv > 0 && ((rc = bind(p.k, a->k, a->k_strides, "k")) || (rc = bind(p.ko, a->k_out, a->ko_strides, "k_out"))))
    return rc;
  p.qw = a->q_weight;
  p.kw = a->k_weight;
  rc = plan_common(pl, a->B, a->T, a->Hq, a->Hkv, a->D, a->rot, a->positions, a->freqs, a->pos_strides, a->sections,
                   a->axes, a->eps, a->dtype, a->param_dtype, a->interleaved != 0, a->q_weight || a->k_weight);
  if (rc) return rc;
  if (p.tokens == 0) return MFX_OK;
  const int64_t blocks = (p.tokens + kWaves - 1) / kWaves;
  pl.grid = dim3((unsigned)blocks, (unsigned)split_heads(pl, p.tokens));
  return MFX_OK;
}

int plan_bwd(const mfx_qk_norm_rope_bwd_args* a, Plan& pl) {
  if (!a) return fail(MFX_E_INVALID, "null args");
  const bool any = a->B != 0 && a->T != 0;
  if (any && ((a->Hq > 0 && (!a->q || !a->dq_out || !a->dq)) || (a->Hkv > 0 && (!a->k || !a->dk_out || !a->dk))))
    return fail(MFX_E_INVALID, "q, dq_out, dq (and with Hkv > 0 k, dk_out, dk) must be non-null");
  Params& p = pl.p;
  int rc = MFX_OK;
  if (a->Hq > 0 && ((rc = bind(p.q, a->q, a->q_strides, "q")) || (rc = bind(p.gq, a->dq_out, a->dqo_strides, "dq_out")) ||
                    (rc = bind(p.qo, a->dq, a->dq_strides, "dq"))))
    return rc;
  if (a->Hkv > 0 && ((rc = bind(p.k, a->k, a->k_strides, "k")) ||
                     (rc = bind(p.gk, a->dk_out, a->dko_strides, "dk_out")) ||
                     (rc = bind(p.ko, a->dk, a->dk_strides, "dk"))))
    return rc;
  p.qw = a->q_weight;
  p.kw = a->k_weight;
  const bool grads = a->dq_weight || a->dk_weight;
  rc = plan_common(pl, a->B, a->T, a->Hq, a->Hkv, a->D, a->rot, a->positions, a->freqs, a->pos_strides, a->sections,
                   a->axes, a->eps, a->dtype, a->param_dtype, a->interleaved != 0,
                   a->q_weight || a->k_weight || grads);
  if (rc) return rc;
  // Workgroups: one token a wavefront up to kMaxPartials of them, then each
  // wavefront walks several (fewer partial rows to add up).
  const int64_t blocks = std::min<int64_t>((p.tokens + kWaves - 1) / kWaves, kMaxPartials);
  const int parts = split_heads(pl, blocks * kWaves);
  pl.grid = dim3((unsigned)std::max<int64_t>(blocks, 1), (unsigned)parts);
  pl.partials = grads && p.tokens > 0 ? (int)blocks * parts : 0;
  return MFX_OK;
}

size_t bwd_bytes(const Plan& pl) { return (size_t)pl.partials * 2 * pl.p.D * sizeof(float); }

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
  if (!pl.partials) return 0;
  // At any alignment: narrower chunks take more lanes a row, hence more parts
  // of the heads, up to one row each or what fills the device (split_heads).
  const int64_t waves = (int64_t)pl.grid.x * mfx::kWaves, want = 8LL * mfx::device_cu_count();
  const int64_t parts = waves < want ? std::min<int64_t>(pl.p.H, (want + waves - 1) / waves) : 1;
  return (size_t)pl.grid.x * parts * 2 * pl.p.D * sizeof(float);
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
  const dim3 grid((unsigned)((2 * pl.p.D + 31) / 32));
  if (pl.f32_params)
    hipLaunchKernelGGL((qk_rope_params<float>), grid, dim3(1024), 0, s, pl.p.partial, pl.partials, pl.p.D,
                       static_cast<float*>(args->dq_weight), static_cast<float*>(args->dk_weight));
  else if (args->dtype == MFX_BF16)
    hipLaunchKernelGGL((qk_rope_params<bf16>), grid, dim3(1024), 0, s, pl.p.partial, pl.partials, pl.p.D,
                       static_cast<bf16*>(args->dq_weight), static_cast<bf16*>(args->dk_weight));
  else
    hipLaunchKernelGGL((qk_rope_params<_Float16>), grid, dim3(1024), 0, s, pl.p.partial, pl.partials, pl.p.D,
                       static_cast<_Float16*>(args->dq_weight), static_cast<_Float16*>(args->dk_weight));
  return launch_status("qk_rope_params");
}

}  // extern "C"

// The norm behind a block, its gate, the residual sum and the norm before the
// next block, one pass over the rows of a residual stream x and a block's
// output y (no counterpart in the reference, whose models leave them to the
// elementwise programs and fast::rms_norm):
//
//   z = y / rms(y) * (o + wp)     (z = y without a norm behind the block)
//   r = alpha x + beta g * z      (g: none, a row for all, for each sequence or each token)
//   h = r / rms(r) * (o + wn)     (of the unrounded r; none without a norm before the next block)
//
// and its gradients, with rh = r / rms(r), u = dh (o + wn), yh = y / rms(y):
//
//   D = dr + (u - rh mean(u rh)) / rms(r),   dx = alpha D
//   dz = beta g D,  v = dz (o + wp),   dy = (v - yh mean(v yh)) / rms(y)
//   dg = beta D z, dwp = dz yh, dwn = dh rh, each summed over the rows that share it
//
// Both are bound by memory: x, y (dr, dh) are read once and r, h (dx, dy) written
// once, a row in the registers of the 64 to 1024 lanes that own it.  Nothing is
// kept from the forward: what the backward needs of it are two more sums over a row
// already in registers.  A group of lanes takes a run of neighbouring rows, so
// that the parameters stay in registers too; the backward's sums over rows
// stay there until the run ends and become one fp32 partial row of the
// workgroup (of a sequence in the group's run for a sequence's gate), which
// residual_params / residual_gates add up in order: no atomics.
#include <algorithm>
#include <cmath>

#include "rowvec.h"
#include "workspace.h"

namespace mfx {
namespace resnorm {
namespace {

using namespace rowvec;

constexpr int VEC = 8;  // elements a lane takes at a time

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct Args {
  const void *x, *y, *gate, *wp, *wn, *dr, *dh;
  void *r, *h, *dx, *dy, *dgate;
  const int32_t* off;
  float* part;       // backward: [workgroups][nsum][ld], then the sequences' slots
  float* slots;      // [groups + sequences][ld]
  int64_t xs, ys, rs, hs, gs, drs, dhs, dxs, dys, dgs, ld;
  int64_t T, S, per;  // rows, sequences, rows of a group
  int H, mode, gate_dt, param_dt;
  int nsum, at_wp, at_wn, at_g;  // which of a workgroup's partial rows (-1: none)
  float alpha, beta, o, post_eps, pre_eps;
};

// VEC values of a row of any of the three types, chosen at run time (uniform).
__device__ __forceinline__ void load_any(const void* p, int dt, int64_t at, int e, int n, float (&out)[VEC]) {
  if (dt == MFX_F32) load_run<float, VEC>(static_cast<const float*>(p) + at, e, n, 0.f, out);
  else if (dt == MFX_BF16) load_run<bf16, VEC>(static_cast<const bf16*>(p) + at, e, n, 0.f, out);
  else load_run<_Float16, VEC>(static_cast<const _Float16*>(p) + at, e, n, 0.f, out);
}
__device__ __forceinline__ void store_any(void* p, int dt, int64_t at, int e, int n, const float (&v)[VEC]) {
  if (dt == MFX_F32) store_run<float, VEC>(static_cast<float*>(p) + at, e, n, v);
  else if (dt == MFX_BF16) store_run<bf16, VEC>(static_cast<bf16*>(p) + at, e, n, v);
  else store_run<_Float16, VEC>(static_cast<_Float16*>(p) + at, e, n, v);
}

// The last sequence that starts at or before token t, 0 if none does.
__device__ __forceinline__ int64_t find_seq(const int32_t* off, int64_t S, int64_t t) {
  int64_t lo = 0, hi = S;  // off[lo] <= t or lo = 0; off[hi] > t or hi = S
  while (hi - lo > 1) {
    const int64_t m = (lo + hi) >> 1;
    if (off[m] <= t) lo = m;
    else hi = m;
  }
  return lo;
}

template <int LANES>
struct Group {
  static constexpr int THREADS = LANES > kBlock ? LANES : kBlock;
  static constexpr int RPB = THREADS / LANES;  // groups of a workgroup
};

// A row's gate in registers: whether the row takes part of y at all, and, for
// a sequence's gate, which sequence's is loaded.
template <int LANES, int NV>
struct Gate {
  float g[NV][VEC];
  int64_t seq = -1, loaded = -1;
  __device__ __forceinline__ void load(const Args& a, int64_t row, int lane) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      load_any(a.gate, a.gate_dt, row * a.gs, (i * LANES + lane) * VEC, a.H, g[i]);
  }
  __device__ __forceinline__ void begin(const Args& a, int64_t t, int lane) {
    if (a.mode == MFX_GATE_FEATURE) load(a, 0, lane);
    if (a.mode == MFX_GATE_NONE) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) g[i][j] = 1.f;
    }
    if (a.mode == MFX_GATE_SEQUENCE && a.S > 0) seq = find_seq(a.off, a.S, t);
  }
  // Row t's gate; false: the row is in no sequence.
  __device__ __forceinline__ bool row(const Args& a, int64_t t, int lane) {
    if (a.mode == MFX_GATE_TOKEN) load(a, t, lane);
    if (a.mode != MFX_GATE_SEQUENCE) return true;
    if (a.S <= 0) return false;
    while (seq + 1 < a.S && a.off[seq + 1] <= t) ++seq;
    if (t < a.off[seq] || t >= a.off[seq + 1]) return false;
    if (seq != loaded) load(a, seq, lane);
    loaded = seq;
    return true;
  }
};

template <int LANES, int NV>
__device__ __forceinline__ void load_weight(const Args& a, const void* w, int lane, float (&out)[NV][VEC]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (w) {
      load_any(w, a.param_dt, 0, (i * LANES + lane) * VEC, a.H, out[i]);
#pragma unroll
      for (int j = 0; j < VEC; ++j) out[i][j] += a.o;
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) out[i][j] = 1.f;
    }
  }
}

template <typename T, int LANES, int NV>
__device__ __forceinline__ void load_row(const void* p, int64_t at, int lane, int n, float (&out)[NV][VEC]) {
#pragma unroll
  for (int i = 0; i < NV; ++i)
    load_run<T, VEC>(static_cast<const T*>(p) + at, (i * LANES + lane) * VEC, n, 0.f, out[i]);
}
template <typename T, int LANES, int NV>
__device__ __forceinline__ void store_row(void* p, int64_t at, int lane, int n, const float (&v)[NV][VEC]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) store_run<T, VEC>(static_cast<T*>(p) + at, (i * LANES + lane) * VEC, n, v[i]);
}

#define FOR_ELEMS                  \
  _Pragma("unroll") for (int i = 0; i < NV; ++i) _Pragma("unroll") for (int j = 0; j < VEC; ++j)

template <typename TX, typename TY, int LANES, int NV>
__global__ __launch_bounds__(Group<LANES>::THREADS) void residual_fwd(Args a) {
  constexpr int RPB = Group<LANES>::RPB;
  __shared__ float lds[Group<LANES>::THREADS / 64];
  const int lane = threadIdx.x % LANES;
  const int64_t grp = (int64_t)blockIdx.x * RPB + threadIdx.x / LANES;
  const int64_t t0 = grp * a.per, t1 = min(a.T, t0 + a.per);
  if (t0 >= t1) return;  // (a whole group; groups of more than a wavefront are workgroups)
  const float inv_n = 1.f / (float)a.H;
  const bool post = a.post_eps >= 0.f, pre = a.pre_eps >= 0.f;
  float wp[NV][VEC], wn[NV][VEC];
  if (post) load_weight<LANES, NV>(a, a.wp, lane, wp);
  if (pre) load_weight<LANES, NV>(a, a.wn, lane, wn);
  Gate<LANES, NV> gate;
  gate.begin(a, t0, lane);
  for (int64_t t = t0; t < t1; ++t) {
    float x[NV][VEC], y[NV][VEC];
    load_row<TX, LANES, NV>(a.x, t * a.xs, lane, a.H, x);
    const bool in = gate.row(a, t, lane);
    load_row<TY, LANES, NV>(a.y, t * a.ys, lane, in ? a.H : 0, y);
    float f = a.beta;
    if (post) {
      float q = 0.f;
      FOR_ELEMS q = fmaf(y[i][j], y[i][j], q);
      const float inv = rsqrtf(row_reduce<LANES, false>(q, lds) * inv_n + a.post_eps);
      f = in ? f * inv : 0.f;
      FOR_ELEMS y[i][j] *= wp[i][j];
    }
    float q = 0.f;
    FOR_ELEMS {
      const float part = in ? f * gate.g[i][j] * y[i][j] : 0.f;
      x[i][j] = fmaf(a.alpha, x[i][j], part);
      q = fmaf(x[i][j], x[i][j], q);
    }
    store_row<TX, LANES, NV>(a.r, t * a.rs, lane, a.H, x);
    if (!pre) continue;
    const float inv = rsqrtf(row_reduce<LANES, false>(q, lds) * inv_n + a.pre_eps);
    FOR_ELEMS x[i][j] *= inv * wn[i][j];
    store_row<TY, LANES, NV>(a.h, t * a.hs, lane, a.H, x);
  }
}

// Adds the groups' sums of a workgroup and writes its partial row k.
template <int LANES, int NV>
__device__ __forceinline__ void write_partial(const Args& a, int k, int lane, int grp, float* fold,
                                              float (&v)[NV][VEC]) {
  constexpr int RPB = Group<LANES>::RPB, W = LANES * NV * VEC;
  if (k < 0) return;
  if constexpr (RPB > 1) {
    __syncthreads();
    FOR_ELEMS fold[grp * W + (i * LANES + lane) * VEC + j] = v[i][j];
    __syncthreads();
    if (grp != 0) return;
#pragma unroll
    for (int b = 1; b < RPB; ++b) FOR_ELEMS v[i][j] += fold[b * W + (i * LANES + lane) * VEC + j];
  }
  store_row<float, LANES, NV>(a.part + ((int64_t)blockIdx.x * a.nsum + k) * a.ld, 0, lane, a.H, v);
}

template <typename TX, typename TY, int LANES, int NV>
__global__ __launch_bounds__(Group<LANES>::THREADS) void residual_bwd(Args a) {
  constexpr int RPB = Group<LANES>::RPB;
  __shared__ float lds[2 * Group<LANES>::THREADS / 64];
  __shared__ float fold[RPB > 1 ? RPB * LANES * NV * VEC : 1];
  const int lane = threadIdx.x % LANES, in_wg = threadIdx.x / LANES;
  const int64_t grp = (int64_t)blockIdx.x * RPB + in_wg;
  const int64_t t0 = min(a.T, grp * a.per), t1 = min(a.T, t0 + a.per);
  const float inv_n = 1.f / (float)a.H;
  const bool post = a.post_eps >= 0.f, pre = a.pre_eps >= 0.f;
  float wp[NV][VEC], wn[NV][VEC], sp[NV][VEC], sn[NV][VEC], sg[NV][VEC];
  FOR_ELEMS sp[i][j] = sn[i][j] = sg[i][j] = 0.f;
  load_weight<LANES, NV>(a, a.wp, lane, wp);
  load_weight<LANES, NV>(a, a.wn, lane, wn);
  Gate<LANES, NV> gate;
  if (t0 < t1) gate.begin(a, t0, lane);
  int64_t cur = -1;  // the sequence whose gate's gradient is in sg
  auto flush = [&]() {
    if (cur >= 0) store_row<float, LANES, NV>(a.slots + (grp + cur) * a.ld, 0, lane, a.H, sg);
    FOR_ELEMS sg[i][j] = 0.f;
  };
  for (int64_t t = t0; t < t1; ++t) {
    float x[NV][VEC], y[NV][VEC], d[NV][VEC], u[NV][VEC];
    load_row<TX, LANES, NV>(a.x, t * a.xs, lane, a.H, x);
    load_row<TX, LANES, NV>(a.dr, t * a.drs, lane, a.dr ? a.H : 0, d);
    load_row<TY, LANES, NV>(a.dh, t * a.dhs, lane, a.dh ? a.H : 0, u);
    const bool in = gate.row(a, t, lane);
    load_row<TY, LANES, NV>(a.y, t * a.ys, lane, in ? a.H : 0, y);
    float iy = 1.f;
    if (post) {
      float q = 0.f;
      FOR_ELEMS q = fmaf(y[i][j], y[i][j], q);
      iy = rsqrtf(row_reduce<LANES, false>(q, lds) * inv_n + a.post_eps);
      FOR_ELEMS y[i][j] = in ? y[i][j] * iy : 0.f;  // yh
    }
    if (pre) {
      float q = 0.f, m = 0.f;
      FOR_ELEMS {
        const float part = in ? a.beta * gate.g[i][j] * (y[i][j] * wp[i][j]) : 0.f;
        x[i][j] = fmaf(a.alpha, x[i][j], part);  // r
        q = fmaf(x[i][j], x[i][j], q);
        m = fmaf(u[i][j] * wn[i][j], x[i][j], m);
      }
      row_reduce_sum2<LANES>(q, m, lds);
      const float ir = rsqrtf(q * inv_n + a.pre_eps);
      const float mr = m * ir * inv_n;
      FOR_ELEMS {
        const float rh = x[i][j] * ir;
        sn[i][j] = fmaf(u[i][j], rh, sn[i][j]);
        d[i][j] = fmaf(ir, u[i][j] * wn[i][j] - rh * mr, d[i][j]);
      }
    }
    // x: dx, u: dy
    FOR_ELEMS x[i][j] = a.alpha * d[i][j];
    store_row<TX, LANES, NV>(a.dx, t * a.dxs, lane, a.H, x);
    if (a.mode == MFX_GATE_SEQUENCE && a.slots && in && gate.seq != cur) {
      flush();
      cur = gate.seq;
    }
    float m = 0.f;
    FOR_ELEMS {
      const float bd = in ? a.beta * d[i][j] : 0.f;
      const float z = y[i][j] * wp[i][j];
      const float dz = in ? bd * gate.g[i][j] : 0.f;
      if (a.mode == MFX_GATE_TOKEN) x[i][j] = bd * z;
      else sg[i][j] = fmaf(bd, z, sg[i][j]);
      u[i][j] = dz;
      if (post) {
        sp[i][j] = fmaf(dz, y[i][j], sp[i][j]);
        u[i][j] = dz * wp[i][j];
        m = fmaf(u[i][j], y[i][j], m);
      }
    }
    if (a.mode == MFX_GATE_TOKEN && a.dgate) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        store_any(a.dgate, a.gate_dt, t * a.dgs, (i * LANES + lane) * VEC, a.H, x[i]);
    }
    if (post) {
      const float my = row_reduce<LANES, false>(m, lds) * inv_n;
      FOR_ELEMS u[i][j] = in ? iy * (u[i][j] - y[i][j] * my) : 0.f;
    }
    store_row<TY, LANES, NV>(a.dy, t * a.dys, lane, a.H, u);
  }
  if (a.mode == MFX_GATE_SEQUENCE && a.slots) flush();
  write_partial<LANES, NV>(a, a.at_wp, lane, in_wg, fold, sp);
  write_partial<LANES, NV>(a, a.at_wn, lane, in_wg, fold, sn);
  write_partial<LANES, NV>(a, a.at_g, lane, in_wg, fold, sg);
}
#undef FOR_ELEMS

// ---- the sums over partial rows ----------------------------------------------------

constexpr int kSumWaves = 16, kSumCols = 64;

// Sum of rows [r0, r1) of p at one column by the WAVES wavefronts of a
// workgroup, in an order that depends on the number of rows alone; valid in
// wavefront 0.
template <int WAVES>
__device__ __forceinline__ float sum_rows(const float* p, int64_t ld, int64_t r0, int64_t r1, int col, int H,
                                          float (&lds)[WAVES][kSumCols]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float s = 0.f;
  if (col < H) {
    constexpr int U = 8;
    for (int64_t r = r0 + wave; r < r1; r += WAVES * U) {
      float v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = r + u * WAVES < r1 ? p[(r + u * WAVES) * ld + col] : 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u) s += v[u];
    }
  }
  lds[wave][lane] = s;
  __syncthreads();
  if (wave == 0)
#pragma unroll
    for (int w = 1; w < WAVES; ++w) s += lds[w][lane];
  return s;
}

__device__ __forceinline__ void store_one(void* p, int dt, int64_t at, float v) {
  if (dt == MFX_F32) static_cast<float*>(p)[at] = v;
  else if (dt == MFX_BF16) static_cast<bf16*>(p)[at] = from_f32<bf16>(v);
  else static_cast<_Float16*>(p)[at] = from_f32<_Float16>(v);
}

struct ParamOut {
  void* p[3];
  int dt[3];
};

// Columns of the gradient k (blockIdx.y): the workgroups' partial rows added.
__global__ __launch_bounds__(kSumWaves * 64) void residual_params(const float* part, int64_t ld, int nsum, int64_t wgs,
                                                                  int H, ParamOut out) {
  __shared__ float lds[kSumWaves][kSumCols];
  const int col = blockIdx.x * kSumCols + (threadIdx.x & 63), k = blockIdx.y;
  const float s = sum_rows<kSumWaves>(part + k * ld, ld * nsum, 0, wgs, col, H, lds);
  if (threadIdx.x < 64 && col < H) store_one(out.p[k], out.dt[k], col, s);
}

// The gradient of sequence blockIdx.y's gate: the slots of the groups whose
// rows are its tokens.  (Group c's slot for sequence s is c + s: going through
// the rows one of them grows at a time, so no two share one.)
template <int WAVES>
__global__ __launch_bounds__(WAVES * 64) void residual_gates(Args a) {
  __shared__ float lds[WAVES][kSumCols];
  const int64_t s = blockIdx.y + (int64_t)blockIdx.z * 65535;
  if (s >= a.S) return;
  const int col = blockIdx.x * kSumCols + (threadIdx.x & 63);
  const int64_t b = max((int64_t)a.off[s], (int64_t)0), e = min((int64_t)a.off[s + 1], a.T);
  int64_t r0 = 0, r1 = 0;
  if (b < e) {
    r0 = b / a.per + s;
    r1 = (e - 1) / a.per + s + 1;
  }
  const float v = sum_rows<WAVES>(a.slots, a.ld, r0, r1, col, a.H, lds);
  if (threadIdx.x < 64 && col < a.H) store_one(a.dgate, a.gate_dt, s * a.dgs + col, v);
}

// ---- host ------------------------------------------------------------------------

bool float_dtype(int dt) { return dt == MFX_F32 || dt == MFX_BF16 || dt == MFX_F16; }

constexpr int64_t kMaxH = 32768;

// Lanes that own a row and their chunks: few lanes leave memory requests in
// flight to few rows, many make the sums over a row dearer.
struct Shape {
  int lanes, nv;
};
Shape shape_of(int64_t H) {
  if (H <= 64 * VEC) return {64, 1};
  if (H <= 128 * VEC) return {64, 2};
  if (H <= 256 * VEC) return {256, 1};
  if (H <= 512 * VEC) return {256, 2};
  if (H <= 1024 * VEC) return {512, 2};
  if (H <= 2048 * VEC) return {1024, 2};
  return {1024, 4};
}

struct Plan {
  Args a{};
  Shape sh{};
  int64_t groups = 0, wgs = 0;
  int res_dtype = 0, dtype = 0, gate_waves = 0;
  ParamOut out{};
  size_t part_bytes = 0, slot_bytes = 0;
};

int bind(const void* p, int64_t stride, int64_t T, int64_t H, int dt, const char* what, bool written) {
  if (!p) return fail(MFX_E_INVALID, std::string(what) + " must be non-null");
  if ((uintptr_t)p % dtype_size(dt)) return fail(MFX_E_INVALID, std::string(what) + " must be aligned to its type");
  if (T > 1 && stride < (written ? H : 0))
    return fail(MFX_E_INVALID, std::string(what) + (written ? ": row stride must be >= H" : ": row stride must be >= 0"));
  return MFX_OK;
}

// What both directions share; groups: as many as `most` of them.
int plan_common(Plan& pl, int64_t T, int64_t H, int64_t S, float alpha, float beta, float o, float post_eps, float pre_eps,
                int res_dtype, int dtype, int param_dtype, int mode, int gate_dtype, const void* x, int64_t xs,
                const void* y, int64_t ys, const void* gate, int64_t gs, const int32_t* off, const void* wp,
                const void* wn, int64_t most) {
  Args& a = pl.a;
  if (T < 0 || H <= 0 || S < 0) return fail(MFX_E_INVALID, "T and num_seqs must be >= 0, H positive");
  if (!float_dtype(res_dtype) || !float_dtype(dtype)) return fail(MFX_E_UNSUPPORTED, "dtypes must be f32, bf16 or f16");
  if (res_dtype != dtype && res_dtype != MFX_F32)
    return fail(MFX_E_UNSUPPORTED, "the residual stream must have the block's type or f32");
  if ((wp || wn) && !float_dtype(param_dtype)) return fail(MFX_E_UNSUPPORTED, "param_dtype must be f32, bf16 or f16");
  if (H > kMaxH) return fail(MFX_E_UNSUPPORTED, "H above 32768 is not supported");
  if (!std::isfinite(alpha) || !std::isfinite(beta) || !std::isfinite(o))
    return fail(MFX_E_INVALID, "alpha, beta and weight_offset must be finite");
  if (!std::isfinite(post_eps) || !std::isfinite(pre_eps))
    return fail(MFX_E_INVALID, "eps must be finite (negative: no norm)");
  if ((wp && post_eps < 0.f) || (wn && pre_eps < 0.f)) return fail(MFX_E_INVALID, "a weight needs its norm (eps >= 0)");
  if (mode < MFX_GATE_NONE || mode > MFX_GATE_TOKEN) return fail(MFX_E_INVALID, "gate_mode must be a MFX_GATE_ value");
  if (mode != MFX_GATE_SEQUENCE && S != 0) return fail(MFX_E_INVALID, "num_seqs belongs to a gate by sequence");
  if (T > 0x7fffffffLL || S > 0x7fffffffLL - 1) return fail(MFX_E_UNSUPPORTED, "problem too large for one launch");
  if (T > 0) {
    if (int rc = bind(x, xs, T, H, res_dtype, "x", false)) return rc;
    if (int rc = bind(y, ys, T, H, dtype, "y", false)) return rc;
  }
  if (mode != MFX_GATE_NONE) {
    if (!float_dtype(gate_dtype)) return fail(MFX_E_UNSUPPORTED, "gate_dtype must be f32, bf16 or f16");
    const int64_t rows = mode == MFX_GATE_FEATURE ? 1 : mode == MFX_GATE_SEQUENCE ? S : T;
    if (rows > 0 && T > 0)
      if (int rc = bind(gate, gs, rows, H, gate_dtype, "gate", false)) return rc;
    if (mode == MFX_GATE_SEQUENCE && (!off || (uintptr_t)off % 4))
      return fail(MFX_E_INVALID, "a gate by sequence needs seq_offsets (4-byte aligned)");
  }
  for (const void* w : {wp, wn})
    if (w && (uintptr_t)w % dtype_size(param_dtype)) return fail(MFX_E_INVALID, "weights must be aligned to their type");
  a.x = x, a.y = y, a.gate = gate, a.wp = wp, a.wn = wn, a.off = off;
  a.xs = xs, a.ys = ys, a.gs = gs;
  a.T = T, a.S = S, a.H = (int)H;
  a.mode = mode, a.gate_dt = gate_dtype, a.param_dt = param_dtype;
  a.alpha = alpha, a.beta = beta, a.o = o, a.post_eps = post_eps, a.pre_eps = pre_eps;
  a.at_wp = a.at_wn = a.at_g = -1;
  pl.sh = shape_of(H);
  pl.res_dtype = res_dtype;
  pl.dtype = dtype;
  if (T == 0) return MFX_OK;
  a.per = ceil_div(T, most);
  const int rpb = pl.sh.lanes < kBlock ? kBlock / pl.sh.lanes : 1;
  pl.groups = ceil_div(T, a.per);
  pl.wgs = ceil_div(pl.groups, rpb);
  return MFX_OK;
}

// f(TX{}, TY{}, lanes, chunks) for the plan's types and shape.
template <int L, int N>
struct Sized {
  static constexpr int lanes = L, nv = N;
};
template <class F, typename TX, typename TY>
void with_shape(const Shape& s, TX x, TY y, F f) {
  if (s.lanes == 64 && s.nv == 1) f(x, y, Sized<64, 1>{});
  else if (s.lanes == 64) f(x, y, Sized<64, 2>{});
  else if (s.lanes == 256 && s.nv == 1) f(x, y, Sized<256, 1>{});
  else if (s.lanes == 256) f(x, y, Sized<256, 2>{});
  else if (s.lanes == 512) f(x, y, Sized<512, 2>{});
  else if (s.nv == 2) f(x, y, Sized<1024, 2>{});
  else f(x, y, Sized<1024, 4>{});
}
template <class F>
void with_kernel(const Plan& pl, F f) {
  if (pl.dtype == MFX_F32) with_shape(pl.sh, float{}, float{}, f);
  else if (pl.dtype == MFX_BF16 && pl.res_dtype == MFX_F32) with_shape(pl.sh, float{}, bf16{}, f);
  else if (pl.dtype == MFX_BF16) with_shape(pl.sh, bf16{}, bf16{}, f);
  else if (pl.res_dtype == MFX_F32) with_shape(pl.sh, float{}, _Float16{}, f);
  else with_shape(pl.sh, _Float16{}, _Float16{}, f);
}

// Groups: what fills the device's wavefront slots (forward) or half of them
// (backward: each workgroup's partial rows cost traffic).
int64_t groups_of(int64_t H, bool bwd) {
  const Shape s = shape_of(H);
  return (int64_t)device_cu_count() * (bwd ? 16 : 32) * 64 / s.lanes;
}

int plan_fwd(const mfx_residual_norm_args* p, Plan& pl) {
  if (!p) return fail(MFX_E_INVALID, "null args");
  const int64_t most = p->H > 0 && p->H <= kMaxH ? groups_of(p->H, false) : 1;
  if (int rc = plan_common(pl, p->T, p->H, p->num_seqs, p->alpha, p->beta, p->weight_offset, p->post_eps, p->pre_eps,
                           p->res_dtype, p->dtype, p->param_dtype, p->gate_mode, p->gate_dtype, p->x, p->x_stride, p->y,
                           p->y_stride, p->gate, p->gate_stride, p->seq_offsets, p->post_weight, p->pre_weight, most))
    return rc;
  if (p->T == 0) return MFX_OK;
  if (int rc = bind(p->r, p->r_stride, p->T, p->H, p->res_dtype, "r", true)) return rc;
  if (p->pre_eps >= 0.f)
    if (int rc = bind(p->h, p->h_stride, p->T, p->H, p->dtype, "h", true)) return rc;
  pl.a.r = p->r, pl.a.h = p->h, pl.a.rs = p->r_stride, pl.a.hs = p->h_stride;
  return MFX_OK;
}

int plan_bwd(const mfx_residual_norm_bwd_args* p, Plan& pl) {
  if (!p) return fail(MFX_E_INVALID, "null args");
  const int64_t most = p->H > 0 && p->H <= kMaxH ? groups_of(p->H, true) : 1;
  if (int rc = plan_common(pl, p->T, p->H, p->num_seqs, p->alpha, p->beta, p->weight_offset, p->post_eps, p->pre_eps,
                           p->res_dtype, p->dtype, p->param_dtype, p->gate_mode, p->gate_dtype, p->x, p->x_stride, p->y,
                           p->y_stride, p->gate, p->gate_stride, p->seq_offsets, p->post_weight, p->pre_weight, most))
    return rc;
  Args& a = pl.a;
  if (p->T > 0 && !p->dr && !p->dh) return fail(MFX_E_INVALID, "dr or dh must be non-null");  // (empty: no address)
  if (p->dh && p->pre_eps < 0.f) return fail(MFX_E_INVALID, "dh belongs to a norm before the next block (pre_eps >= 0)");
  if ((p->dpost_weight && !p->post_weight) || (p->dpre_weight && !p->pre_weight) ||
      (p->dgate && p->gate_mode == MFX_GATE_NONE))
    return fail(MFX_E_INVALID, "a gradient needs its weight or gate");
  for (const void* w : {p->dpost_weight, p->dpre_weight})
    if (w && (uintptr_t)w % dtype_size(p->param_dtype))
      return fail(MFX_E_INVALID, "gradients must be aligned to their type");
  if (p->dgate) {
    const int64_t rows = p->gate_mode == MFX_GATE_FEATURE ? 1 : p->gate_mode == MFX_GATE_SEQUENCE ? p->num_seqs : p->T;
    if (rows > 0)
      if (int rc = bind(p->dgate, p->dgate_stride, rows, p->H, p->gate_dtype, "dgate", true)) return rc;
  }
  if (p->T > 0) {
    if (p->dr)
      if (int rc = bind(p->dr, p->dr_stride, p->T, p->H, p->res_dtype, "dr", false)) return rc;
    if (p->dh)
      if (int rc = bind(p->dh, p->dh_stride, p->T, p->H, p->dtype, "dh", false)) return rc;
    if (int rc = bind(p->dx, p->dx_stride, p->T, p->H, p->res_dtype, "dx", true)) return rc;
    if (int rc = bind(p->dy, p->dy_stride, p->T, p->H, p->dtype, "dy", true)) return rc;
  }
  a.dr = p->dr, a.dh = p->dh, a.dx = p->dx, a.dy = p->dy, a.dgate = p->dgate;
  a.drs = p->dr_stride, a.dhs = p->dh_stride, a.dxs = p->dx_stride, a.dys = p->dy_stride, a.dgs = p->dgate_stride;
  a.ld = ceil_div(p->H, VEC) * VEC;
  auto sum = [&](void* to, int dt, int& at) {
    if (!to) return;
    pl.out.p[a.nsum] = to;
    pl.out.dt[a.nsum] = dt;
    at = a.nsum++;
  };
  sum(p->dpost_weight, p->param_dtype, a.at_wp);
  sum(p->dpre_weight, p->param_dtype, a.at_wn);
  if (p->gate_mode == MFX_GATE_FEATURE) sum(p->dgate, p->gate_dtype, a.at_g);
  pl.part_bytes = align256((size_t)pl.wgs * a.nsum * a.ld * 4);
  // (Groups that the last workgroup has beyond the last rows' write no slot.)
  if (p->gate_mode == MFX_GATE_SEQUENCE && p->dgate && p->num_seqs > 0) {
    pl.slot_bytes = (size_t)(pl.groups + p->num_seqs) * a.ld * 4;
    // (Short sequences have a few slots each, a wavefront's work.)
    pl.gate_waves = pl.groups < 16 * p->num_seqs ? 1 : kSumWaves;
    if (!launch_fits(ceil_div(p->H, kSumCols) * p->num_seqs, pl.gate_waves * 64))
      return fail(MFX_E_UNSUPPORTED, "problem too large for one launch");
  }
  return MFX_OK;
}

}  // namespace
}  // namespace resnorm
}  // namespace mfx

extern "C" {

int mfx_residual_norm(const mfx_residual_norm_args* args, void* stream) {
  using namespace mfx;
  using namespace mfx::resnorm;
  Plan pl;
  if (int rc = plan_fwd(args, pl)) return rc;
  if (args->T == 0) return MFX_OK;
  with_kernel(pl, [&](auto tx, auto ty, auto sz) {
    typedef decltype(sz) Z;
    hipLaunchKernelGGL((residual_fwd<decltype(tx), decltype(ty), Z::lanes, Z::nv>), dim3((unsigned)pl.wgs),
                       dim3(Group<Z::lanes>::THREADS), 0, static_cast<hipStream_t>(stream), pl.a);
  });
  return launch_status("residual_fwd");
}

size_t mfx_residual_norm_bwd_workspace_size(const mfx_residual_norm_bwd_args* args) {
  mfx::resnorm::Plan pl;
  return mfx::resnorm::plan_bwd(args, pl) == MFX_OK ? pl.part_bytes + pl.slot_bytes : 0;
}

int mfx_residual_norm_bwd(const mfx_residual_norm_bwd_args* args, void* stream) {
  using namespace mfx;
  using namespace mfx::resnorm;
  Plan pl;
  if (int rc = plan_bwd(args, pl)) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  Args& a = pl.a;
  char* ws = nullptr;
  if (int rc = take_workspace(args->workspace, args->workspace_bytes, pl.part_bytes + pl.slot_bytes,
                              "mfx_residual_norm_bwd_workspace_size", s, &ws))
    return rc;
  a.part = reinterpret_cast<float*>(ws);
  a.slots = pl.slot_bytes ? reinterpret_cast<float*>(ws + pl.part_bytes) : nullptr;
  if (a.T > 0) {
    with_kernel(pl, [&](auto tx, auto ty, auto sz) {
      typedef decltype(sz) Z;
      hipLaunchKernelGGL((residual_bwd<decltype(tx), decltype(ty), Z::lanes, Z::nv>), dim3((unsigned)pl.wgs),
                         dim3(Group<Z::lanes>::THREADS), 0, s, a);
    });
    if (int rc = launch_status("residual_bwd")) return rc;
  }
  const unsigned cols = (unsigned)ceil_div(a.H, kSumCols);
  if (a.nsum) {
    hipLaunchKernelGGL(residual_params, dim3(cols, a.nsum), dim3(kSumWaves * 64), 0, s, a.part, a.ld, a.nsum, pl.wgs,
                       a.H, pl.out);
    if (int rc = launch_status("residual_params")) return rc;
  }
  if (a.mode == MFX_GATE_SEQUENCE && a.dgate && a.S > 0) {
    const int64_t y = std::min<int64_t>(a.S, 65535), z = ceil_div(a.S, 65535);
    const dim3 grid(cols, (unsigned)y, (unsigned)z);
    if (pl.gate_waves == 1) hipLaunchKernelGGL((residual_gates<1>), grid, dim3(64), 0, s, a);
    else hipLaunchKernelGGL((residual_gates<kSumWaves>), grid, dim3(kSumWaves * 64), 0, s, a);
    return launch_status("residual_gates");
  }
  return MFX_OK;
}

}  // extern "C"

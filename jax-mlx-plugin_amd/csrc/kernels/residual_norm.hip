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
//
// Measured: 8192 rows of 4096 in bf16 forward 46 us (5.9 TB/s, with the call), backward with the
// stream in f32 and both norms 123 us and 5 for the weights (5.0 TB/s, a copy's rate); 4099 of
// 2048 with a gate backward 25 and 4.  Rows of up to 1536 with a gate and both norms wait for
// their three sums: 8192 of 1536 backward 54 us with the call (2.8 TB/s).  64 rows of 4096 take 4 us.
// Rows of over 8192 (and, by less, gated and odd ones of over 4096) spill registers in the
// backward: 2048 of 16384 528 us (0.8 TB/s).
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

// A lane's VEC elements of a row as they come, so that loads stay in flight: no
// branch and no use between one load and the next (a load of a row's whole chunks
// beside one of its last elements, each unpacked on the spot, waited for every tensor
// of a row in turn: 155 us for 8192 rows of 4096 backward).  A lane past the row's
// end reads its last VEC elements again.  Of a row that is not whole chunks (not
// EASY) its last lane does so too and shifts what it needs down, zeros behind it.
template <typename T, bool EASY>
struct Raw {
  static constexpr int N = VEC * sizeof(T) / 4;
  uint32_t w[N];
  __device__ __forceinline__ void load(const void* p, int64_t at, int e, int n) {
    if (EASY || n >= VEC) {
      typedef uint32_t run_t __attribute__((ext_vector_type(4), aligned(2)));
      const T* from = static_cast<const T*>(p) + at + min(e, n - VEC);
#pragma unroll
      for (int c = 0; c < N / 4; ++c) {
        const run_t r = reinterpret_cast<const run_t*>(from)[c];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[c * 4 + j] = r[j];
      }
    } else {  // a row shorter than a chunk, the same for all lanes
#pragma unroll
      for (int j = 0; j < N; ++j) w[j] = 0;
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (e == 0 && j < n) {
          if constexpr (sizeof(T) == 4) w[j] = static_cast<const uint32_t*>(p)[at + j];
          else w[j / 2] |= (uint32_t)static_cast<const uint16_t*>(p)[at + j] << (16 * (j & 1));
        }
    }
  }
  // Elements of the row from e on (EASY: any where e lies past its end).
  __device__ __forceinline__ void get(int e, int n, float (&out)[VEC]) const {
    uint32_t x[N];
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = w[j];
    if (!EASY && n >= VEC) {
      const int s = max(0, min(VEC, e + VEC - n));  // elements to shift down by
      const int words = sizeof(T) == 4 ? s : s >> 1;
#pragma unroll
      for (int step = 1; step <= N; step *= 2)
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = words & step ? (j + step < N ? x[j + step] : 0u) : x[j];
      if constexpr (sizeof(T) == 2)
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = s & 1 ? x[j] >> 16 | (j + 1 < N ? x[j + 1] << 16 : 0u) : x[j];
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) out[j] = __uint_as_float(x[j]);
    } else {
      unpack16<T>(make_uint4(x[0], x[1], x[2], x[3]), out);
    }
  }
};

// The same of a tensor of any of the three types, chosen at run time (uniform).
template <bool EASY>
struct RawAny {
  Raw<float, EASY> f;  // (of a 16-bit tensor the first half)
  __device__ __forceinline__ void load(const void* p, int dt, int64_t at, int e, int n) {
    if (dt == MFX_F32) return f.load(p, at, e, n);
    Raw<bf16, EASY> h;
    h.load(p, at, e, n);
#pragma unroll
    for (int j = 0; j < h.N; ++j) f.w[j] = h.w[j];
  }
  template <typename T>
  __device__ __forceinline__ void get16(int e, int n, float (&out)[VEC]) const {
    Raw<T, EASY> h;
#pragma unroll
    for (int j = 0; j < h.N; ++j) h.w[j] = f.w[j];
    h.get(e, n, out);
  }
  __device__ __forceinline__ void get(int dt, int e, int n, float (&out)[VEC]) const {
    if (dt == MFX_F32) f.get(e, n, out);
    else if (dt == MFX_BF16) get16<bf16>(e, n, out);
    else get16<_Float16>(e, n, out);
  }
};

// A chunk's elements of a row; EASY rows have no last, partial one.
template <typename T, bool EASY>
__device__ __forceinline__ void store_chunk(void* p, int64_t at, int e, int n, const float (&v)[VEC]) {
  T* const row = static_cast<T*>(p) + at;
  if constexpr (EASY) {
    if (e < n) store_run<T, VEC>(row, e, e + VEC, v);
  } else {
    store_run<T, VEC>(row, e, n, v);
  }
}

template <bool EASY>
__device__ __forceinline__ void store_any(void* p, int dt, int64_t at, int e, int n, const float (&v)[VEC]) {
  if (dt == MFX_F32) store_chunk<float, EASY>(p, at, e, n, v);
  else if (dt == MFX_BF16) store_chunk<bf16, EASY>(p, at, e, n, v);
  else store_chunk<_Float16, EASY>(p, at, e, n, v);
}

// The last sequence that starts at or before token t, 0 if none does: 64 offsets at
// a time, a lane each.  All lanes of a wavefront look for tokens of their own group.
__device__ __forceinline__ int64_t find_seq(const int32_t* off, int64_t S, int64_t t) {
  int64_t lo = 0, n = S;  // among the n from lo on
  while (n > 1) {
    const int64_t step = (n + 63) / 64;
    const int64_t i = lo + (threadIdx.x & 63) * step;
    const uint64_t at = __ballot(i < lo + n && off[min(i, S)] <= t);
    // (Offsets ascend: the lanes that say so are the first ones.)
    const int hits = (int)__popcll(at), last = hits > 0 ? hits - 1 : 0;
    n = min(step, n - last * step);
    lo += last * step;
  }
  return lo;
}

// What a gate's rows are shared by: kNone no gate, kShared one row, or one a
// sequence, kToken one a token, kAny any of them, decided at run time.
enum Kind { kNone, kShared, kToken, kAny };

template <int LANES>
struct Group {
  static constexpr int THREADS = LANES > 64 ? LANES : kBlock;
  static constexpr int RPB = THREADS / LANES;  // groups of a workgroup
};

#define FOR_CHUNKS _Pragma("unroll") for (int i = 0; i < NV; ++i)
#define FOR_ELEMS FOR_CHUNKS _Pragma("unroll") for (int j = 0; j < VEC; ++j)

// A lane's chunks of a row: elements (i * LANES + lane) * VEC and on.
template <int LANES_, int NV_, bool EASY_>
struct Place {
  static constexpr int LANES = LANES_, NV = NV_;
  static constexpr bool EASY = EASY_;
  int lane, n;
  bool in[NV];  // any of the chunk lies in the row
  __device__ __forceinline__ Place(int H) : lane(threadIdx.x % LANES), n(H) {
    FOR_CHUNKS in[i] = e(i) < n;
  }
  __device__ __forceinline__ int e(int i) const { return (i * LANES + lane) * VEC; }
  template <typename T>
  __device__ __forceinline__ void load(Raw<T, EASY> (&r)[NV], const void* p, int64_t at) const {
    FOR_CHUNKS r[i].load(p, at, e(i), n);
  }
  template <typename T>
  __device__ __forceinline__ void get(const Raw<T, EASY> (&r)[NV], float (&out)[NV][VEC]) const {
    FOR_CHUNKS r[i].get(e(i), n, out[i]);
  }
  template <typename T>
  __device__ __forceinline__ void store(void* p, int64_t at, const float (&v)[NV][VEC]) const {
    FOR_CHUNKS store_chunk<T, EASY>(p, at, e(i), n, v[i]);
  }
  // Sum over the row of f(i, j, so far) (lanes past its end add nothing).
  template <class F>
  __device__ __forceinline__ float sum(F f) const {
    float s = 0.f;
    FOR_CHUNKS {
      float c = 0.f;
#pragma unroll
      for (int j = 0; j < VEC; ++j) c = f(i, j, c);
      s += in[i] ? c : 0.f;
    }
    return s;
  }
};

template <class P>
__device__ __forceinline__ void load_weight(const Args& a, const P& at, const void* w, float (&out)[P::NV][VEC]) {
  constexpr int NV = P::NV;
  FOR_ELEMS out[i][j] = 1.f;
  if (!w) return;
  FOR_CHUNKS {
    RawAny<P::EASY> r;
    r.load(w, a.param_dt, 0, at.e(i), at.n);
    r.get(a.param_dt, at.e(i), at.n, out[i]);
  }
  FOR_ELEMS out[i][j] += a.o;
}

// The gate of a group's rows: the one row of all, or the row's sequence's (whose
// row is loaded when it changes) or its own.
template <class P, Kind KIND>
struct Gate {
  static constexpr int NV = P::NV;
  float g[NV][VEC];
  RawAny<P::EASY> next[NV];  // of a gate by token: the next row's
  int64_t seq = -1;
  int32_t first = 0, end = 0;  // its tokens
  __device__ __forceinline__ bool token(const Args& a) const {
    return KIND == kToken || (KIND == kAny && a.mode == MFX_GATE_TOKEN);
  }
  __device__ __forceinline__ bool sequence(const Args& a) const {
    return (KIND == kShared || KIND == kAny) && a.mode == MFX_GATE_SEQUENCE;
  }
  __device__ __forceinline__ void take(const Args& a, const P& at) {
    FOR_CHUNKS next[i].get(a.gate_dt, at.e(i), at.n, g[i]);
  }
  __device__ __forceinline__ void fetch(const Args& a, const P& at, int64_t row) {
    FOR_CHUNKS next[i].load(a.gate, a.gate_dt, row * a.gs, at.e(i), at.n);
  }
  __device__ __forceinline__ void turn(const Args& a, const P& at) {
    first = a.off[seq];
    end = a.off[seq + 1];
    fetch(a, at, seq);
    take(a, at);
  }
  __device__ __forceinline__ void begin(const Args& a, const P& at, int64_t t) {
    FOR_ELEMS g[i][j] = 1.f;
    if (token(a)) {
      fetch(a, at, t);
    } else if (sequence(a)) {
      if (a.S <= 0) return;
      seq = find_seq(a.off, a.S, t);
      turn(a, at);
    } else if (KIND == kShared || a.mode == MFX_GATE_FEATURE) {
      fetch(a, at, 0);
      take(a, at);
    }
  }
  // Row t's gate, and the fetch of row `after`'s; false: the row is in no sequence.
  __device__ __forceinline__ bool row(const Args& a, const P& at, int64_t t, int64_t after) {
    if (token(a)) {
      take(a, at);
      fetch(a, at, after);
    }
    if (!sequence(a)) return true;
    if (a.S <= 0) return false;
    if (t >= end && seq + 1 < a.S && a.off[seq + 1] <= t) {
      do ++seq;
      while (seq + 1 < a.S && a.off[seq + 1] <= t);
      turn(a, at);
    }
    return t >= first && t < end;
  }
};

template <typename TX, typename TY, class P, Kind KIND>
__global__ __launch_bounds__(Group<P::LANES>::THREADS) void residual_fwd(Args a) {
  constexpr int LANES = P::LANES, NV = P::NV, RPB = Group<LANES>::RPB;
  constexpr bool GATED = KIND != kNone;
  __shared__ float lds[Group<LANES>::THREADS / 64];
  const P at(a.H);
  const int64_t grp = (int64_t)blockIdx.x * RPB + threadIdx.x / LANES;
  const int64_t t0 = grp * a.per, t1 = min(a.T, t0 + a.per);
  if (t0 >= t1) return;  // (a whole group; groups of more than a wavefront are workgroups)
  const float inv_n = 1.f / (float)a.H;
  const bool post = a.post_eps >= 0.f, pre = a.pre_eps >= 0.f;
  Raw<TX, P::EASY> xr[NV];
  Raw<TY, P::EASY> yr[NV];
  at.load(yr, a.y, t0 * a.ys);
  at.load(xr, a.x, t0 * a.xs);
  float wp[NV][VEC], wn[NV][VEC];
  load_weight(a, at, a.wp, wp);
  load_weight(a, at, a.wn, wn);
  Gate<P, KIND> gate;
  if (GATED) gate.begin(a, at, t0);
  for (int64_t t = t0; t < t1; ++t) {
    float x[NV][VEC], y[NV][VEC];
    at.get(yr, y);
    at.get(xr, x);
    const int64_t next = min(t + 1, t1 - 1);
    if (t + 1 < t1) {
      at.load(yr, a.y, next * a.ys);
      at.load(xr, a.x, next * a.xs);
    }
    const bool in = !GATED || gate.row(a, at, t, next);
    float f = a.beta;
    if (post) {
      const float q = at.sum([&](int i, int j, float s) { return fmaf(y[i][j], y[i][j], s); });
      f *= rsqrtf(row_reduce<LANES, false>(q, lds) * inv_n + a.post_eps);
      FOR_ELEMS y[i][j] *= wp[i][j];
    }
    FOR_ELEMS {
      if (GATED) x[i][j] = fmaf(a.alpha, x[i][j], in ? f * gate.g[i][j] * y[i][j] : 0.f);
      else x[i][j] = fmaf(a.alpha, x[i][j], f * y[i][j]);
    }
    at.template store<TX>(a.r, t * a.rs, x);
    if (!pre) continue;
    const float q = at.sum([&](int i, int j, float s) { return fmaf(x[i][j], x[i][j], s); });
    const float inv = rsqrtf(row_reduce<LANES, false>(q, lds) * inv_n + a.pre_eps);
    FOR_ELEMS x[i][j] *= inv * wn[i][j];
    at.template store<TY>(a.h, t * a.hs, x);
  }
}

// Adds the groups' sums of a workgroup and writes its partial row k.
template <class P>
__device__ __forceinline__ void write_partial(const Args& a, const P& at, int k, int grp, float* fold,
                                              float (&v)[P::NV][VEC]) {
  constexpr int NV = P::NV, RPB = Group<P::LANES>::RPB, W = P::LANES * NV * VEC;
  if (k < 0) return;
  if constexpr (RPB > 1) {
    __syncthreads();
    FOR_ELEMS fold[grp * W + at.e(i) + j] = v[i][j];
    __syncthreads();
    if (grp != 0) return;
#pragma unroll
    for (int b = 1; b < RPB; ++b) FOR_ELEMS v[i][j] += fold[b * W + at.e(i) + j];
  }
  at.template store<float>(a.part + ((int64_t)blockIdx.x * a.nsum + k) * a.ld, 0, v);
}

template <typename TX, typename TY, class P, Kind KIND>
__global__ __launch_bounds__(Group<P::LANES>::THREADS) void residual_bwd(Args a) {
  constexpr int LANES = P::LANES, NV = P::NV, RPB = Group<LANES>::RPB;
  constexpr bool GATED = KIND != kNone;
  __shared__ float lds[2 * Group<LANES>::THREADS / 64];
  __shared__ float fold[RPB > 1 ? RPB * LANES * NV * VEC : 1];
  const P at(a.H);
  const int in_wg = threadIdx.x / LANES;
  const int64_t grp = (int64_t)blockIdx.x * RPB + in_wg;
  const int64_t t0 = min(a.T, grp * a.per), t1 = min(a.T, t0 + a.per);
  const float inv_n = 1.f / (float)a.H;
  const bool post = a.post_eps >= 0.f, pre = a.pre_eps >= 0.f;
  float sp[NV][VEC], sn[NV][VEC], sg[NV][VEC];
  FOR_ELEMS sp[i][j] = sn[i][j] = sg[i][j] = 0.f;
  if (t0 < t1) {
    Raw<TX, P::EASY> xr[NV], dr[NV];
    Raw<TY, P::EASY> yr[NV], ur[NV];
    // (Without a gradient: x or y in its place, not used.)
    const void* const dh = a.dh ? a.dh : a.y;
    const void* const up = a.dr ? a.dr : a.x;
    const int64_t us = a.dh ? a.dhs : a.ys, ds = a.dr ? a.drs : a.xs;
    auto fetch = [&](int64_t t) __attribute__((always_inline)) {
      at.load(yr, a.y, t * a.ys);
      at.load(xr, a.x, t * a.xs);
      at.load(ur, dh, t * us);
      at.load(dr, up, t * ds);
    };
    fetch(t0);
    float wp[NV][VEC], wn[NV][VEC];
    load_weight(a, at, a.wp, wp);
    load_weight(a, at, a.wn, wn);
    Gate<P, KIND> gate;
    if (GATED) gate.begin(a, at, t0);
    int64_t cur = -1;  // the sequence whose gate's gradient is in sg
    auto flush = [&]() {
      if (cur >= 0) at.template store<float>(a.slots + (grp + cur) * a.ld, 0, sg);
      FOR_ELEMS sg[i][j] = 0.f;
    };
    for (int64_t t = t0; t < t1; ++t) {
      float x[NV][VEC], y[NV][VEC], d[NV][VEC], u[NV][VEC];
      at.get(yr, y);
      at.get(xr, x);
      at.get(ur, u);
      at.get(dr, d);
      if (!a.dh) FOR_ELEMS u[i][j] = 0.f;
      if (!a.dr) FOR_ELEMS d[i][j] = 0.f;
      if (t + 1 < t1) fetch(t + 1);
      const bool in = !GATED || gate.row(a, at, t, min(t + 1, t1 - 1));
      float iy = 1.f;
      if (post) {
        const float q = at.sum([&](int i, int j, float s) { return fmaf(y[i][j], y[i][j], s); });
        iy = rsqrtf(row_reduce<LANES, false>(q, lds) * inv_n + a.post_eps);
        FOR_ELEMS y[i][j] *= iy;  // yh
      }
      if (GATED && !in) FOR_ELEMS y[i][j] = 0.f;
      if (pre) {
        FOR_ELEMS {
          const float z = y[i][j] * wp[i][j];
          x[i][j] = fmaf(a.alpha, x[i][j], a.beta * (GATED ? (in ? gate.g[i][j] * z : 0.f) : z));  // r
        }
        float q = at.sum([&](int i, int j, float s) { return fmaf(x[i][j], x[i][j], s); });
        float m = at.sum([&](int i, int j, float s) { return fmaf(u[i][j] * wn[i][j], x[i][j], s); });
        row_reduce_sum2<LANES>(q, m, lds);
        const float ir = rsqrtf(q * inv_n + a.pre_eps);
        const float mr = m * ir * inv_n;
        FOR_ELEMS {
          const float rh = x[i][j] * ir;
          sn[i][j] = fmaf(u[i][j], rh, sn[i][j]);
          d[i][j] = fmaf(ir, u[i][j] * wn[i][j] - rh * mr, d[i][j]);
        }
      }
      FOR_ELEMS x[i][j] = a.alpha * d[i][j];
      at.template store<TX>(a.dx, t * a.dxs, x);
      // u: dz, then dy
      FOR_ELEMS u[i][j] = a.beta * d[i][j];
      if constexpr (GATED) {
        if (gate.sequence(a) && a.slots && in && gate.seq != cur) {
          flush();
          cur = gate.seq;
        }
        if (!in) FOR_ELEMS u[i][j] = 0.f;
        if (gate.token(a)) {
          FOR_ELEMS x[i][j] = u[i][j] * (y[i][j] * wp[i][j]);
          if (a.dgate) FOR_CHUNKS store_any<P::EASY>(a.dgate, a.gate_dt, t * a.dgs, at.e(i), at.n, x[i]);
        } else {
          FOR_ELEMS sg[i][j] = fmaf(u[i][j], y[i][j] * wp[i][j], sg[i][j]);
        }
        if (in) FOR_ELEMS u[i][j] *= gate.g[i][j];
      }
      if (post) {
        FOR_ELEMS {
          sp[i][j] = fmaf(u[i][j], y[i][j], sp[i][j]);
          u[i][j] *= wp[i][j];
        }
        const float m = at.sum([&](int i, int j, float s) { return fmaf(u[i][j], y[i][j], s); });
        const float my = row_reduce<LANES, false>(m, lds) * inv_n;
        FOR_ELEMS u[i][j] = GATED && !in ? 0.f : iy * (u[i][j] - y[i][j] * my);
      }
      at.template store<TY>(a.dy, t * a.dys, u);
    }
    if (GATED && gate.sequence(a) && a.slots) flush();
  }
  write_partial(a, at, a.at_wp, in_wg, fold, sp);
  write_partial(a, at, a.at_wn, in_wg, fold, sn);
  if (KIND == kShared || KIND == kAny) write_partial(a, at, a.at_g, in_wg, fold, sg);
}
#undef FOR_ELEMS
#undef FOR_CHUNKS

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

// Lanes that own a row and their chunks: a chunk a lane, of lanes that leave few
// idle, while the lanes have registers for the backward (its 4096 rows of 5120 take 58 us
// in 768 lanes for 70 in 1024; of 8192 with a gate 126 us in 512 lanes of two chunks for 156, of
// 6144 89 for 184).  Rows that are not whole chunks, whose shifts take registers too, have a
// chunk a lane while there are lanes (5001: 109 us in 768, 234 in 1024, 371 in 512 of two).
struct Shape {
  int lanes, nv;
  bool easy;
};
Shape shape_of(int64_t H) {
  const bool easy = H % VEC == 0;
  const int64_t chunks = ceil_div(H, VEC);
  for (int lanes : {64, 128, 192, 256, 384, 512, 768}) {
    if (chunks <= lanes) return {lanes, 1, easy};
  }
  if (chunks <= 1024) return easy ? Shape{512, 2, true} : Shape{1024, 1, false};
  return {1024, chunks <= 2048 && easy ? 2 : 4, easy};
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

int64_t groups_of(int64_t H, bool bwd);

// What both directions share.
int plan_common(Plan& pl, int64_t T, int64_t H, int64_t S, float alpha, float beta, float o, float post_eps, float pre_eps,
                int res_dtype, int dtype, int param_dtype, int mode, int gate_dtype, const void* x, int64_t xs,
                const void* y, int64_t ys, const void* gate, int64_t gs, const int32_t* off, const void* wp,
                const void* wn, bool bwd) {
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
  a.per = ceil_div(T, groups_of(H, bwd));
  const int rpb = pl.sh.lanes <= 64 ? kBlock / pl.sh.lanes : 1;
  pl.groups = ceil_div(T, a.per);
  pl.wgs = ceil_div(pl.groups, rpb);
  return MFX_OK;
}

// f(TX{}, TY{}, a Place, a Kind) for the plan's types and shape.
template <int L, int N, bool E>
struct Sized {
  typedef Place<L, N, E> P;
};
template <Kind K>
using KindOf = std::integral_constant<Kind, K>;
template <class F, typename TX, typename TY>
void with_shape(const Plan& pl, TX x, TY y, F f) {
  const Shape& s = pl.sh;
  if (!s.easy) {
    const KindOf<kAny> k;
    if (s.lanes == 64) f(x, y, Sized<64, 1, false>{}, k);
    else if (s.lanes == 128) f(x, y, Sized<128, 1, false>{}, k);
    else if (s.lanes == 192) f(x, y, Sized<192, 1, false>{}, k);
    else if (s.lanes == 256) f(x, y, Sized<256, 1, false>{}, k);
    else if (s.lanes == 384) f(x, y, Sized<384, 1, false>{}, k);
    else if (s.lanes == 512) f(x, y, Sized<512, 1, false>{}, k);
    else if (s.lanes == 768) f(x, y, Sized<768, 1, false>{}, k);
    else if (s.nv == 1) f(x, y, Sized<1024, 1, false>{}, k);
    else f(x, y, Sized<1024, 4, false>{}, k);
    return;
  }
  if (s.lanes == 1024) {
    const KindOf<kAny> k;
    if (s.nv == 2) f(x, y, Sized<1024, 2, true>{}, k);
    else f(x, y, Sized<1024, 4, true>{}, k);
    return;
  }
  auto kind = [&](auto k) {
    if (s.lanes == 64) f(x, y, Sized<64, 1, true>{}, k);
    else if (s.lanes == 128) f(x, y, Sized<128, 1, true>{}, k);
    else if (s.lanes == 192) f(x, y, Sized<192, 1, true>{}, k);
    else if (s.lanes == 256) f(x, y, Sized<256, 1, true>{}, k);
    else if (s.lanes == 384) f(x, y, Sized<384, 1, true>{}, k);
    else if (s.lanes == 768) f(x, y, Sized<768, 1, true>{}, k);
    else if (s.nv == 1) f(x, y, Sized<512, 1, true>{}, k);
    else f(x, y, Sized<512, 2, true>{}, k);
  };
  if (pl.a.mode == MFX_GATE_NONE) kind(KindOf<kNone>{});
  else if (pl.a.mode == MFX_GATE_TOKEN) kind(KindOf<kToken>{});
  else kind(KindOf<kShared>{});
}
template <class F>
void with_kernel(const Plan& pl, F f) {
  if (pl.dtype == MFX_F32) with_shape(pl, float{}, float{}, f);
  else if (pl.dtype == MFX_BF16 && pl.res_dtype == MFX_F32) with_shape(pl, float{}, bf16{}, f);
  else if (pl.dtype == MFX_BF16) with_shape(pl, bf16{}, bf16{}, f);
  else if (pl.res_dtype == MFX_F32) with_shape(pl, float{}, _Float16{}, f);
  else with_shape(pl, _Float16{}, _Float16{}, f);
}

// Groups: 16 wavefronts a CU (forward) or 8 (backward, where each workgroup's partial
// rows cost traffic; 12 of rows that two or three own, whose sums leave them waiting for
// each other: 16384 rows of 1024 with a gate 50 us for 54, 4099 of 1152 32 for 35), and a
// workgroup a CU at least.
int64_t groups_of(int64_t H, bool bwd) {
  const int lanes = shape_of(H).lanes, waves = !bwd ? 16 : lanes == 128 || lanes == 192 ? 12 : 8;
  return (int64_t)device_cu_count() * std::max(1, waves * 64 / lanes);
}

int plan_fwd(const mfx_residual_norm_args* p, Plan& pl) {
  if (!p) return fail(MFX_E_INVALID, "null args");
  if (int rc = plan_common(pl, p->T, p->H, p->num_seqs, p->alpha, p->beta, p->weight_offset, p->post_eps, p->pre_eps,
                           p->res_dtype, p->dtype, p->param_dtype, p->gate_mode, p->gate_dtype, p->x, p->x_stride, p->y,
                           p->y_stride, p->gate, p->gate_stride, p->seq_offsets, p->post_weight, p->pre_weight, false))
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
  if (int rc = plan_common(pl, p->T, p->H, p->num_seqs, p->alpha, p->beta, p->weight_offset, p->post_eps, p->pre_eps,
                           p->res_dtype, p->dtype, p->param_dtype, p->gate_mode, p->gate_dtype, p->x, p->x_stride, p->y,
                           p->y_stride, p->gate, p->gate_stride, p->seq_offsets, p->post_weight, p->pre_weight, true))
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
  with_kernel(pl, [&](auto tx, auto ty, auto sz, auto k) {
    typedef typename decltype(sz)::P P;
    hipLaunchKernelGGL((residual_fwd<decltype(tx), decltype(ty), P, decltype(k)::value>), dim3((unsigned)pl.wgs),
                       dim3(Group<P::LANES>::THREADS), 0, static_cast<hipStream_t>(stream), pl.a);
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
    with_kernel(pl, [&](auto tx, auto ty, auto sz, auto k) {
      typedef typename decltype(sz)::P P;
      hipLaunchKernelGGL((residual_bwd<decltype(tx), decltype(ty), P, decltype(k)::value>), dim3((unsigned)pl.wgs),
                         dim3(Group<P::LANES>::THREADS), 0, s, a);
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

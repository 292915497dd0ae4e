// Embedding lookup and the gradient of its table (no counterpart in the
// reference, whose models take embedded inputs):
//
//   out[t] = scale * w[ids[t]]              (zeros for an id outside [0, V))
//   dw[v]  = [dw[v] +] scale * sum over t with ids[t] = v of dout[t]
//
// Both are bound by memory: the forward reads and writes T rows, the backward
// reads T rows and writes V.  Sums are fp32, each output rounded once.
//
// The backward sorts the tokens by id, so that each row of dw is written once,
// by one owner, without atomics, its tokens added in their order:
//   embed_index  Each workgroup owns a run of up to 480 rows of the table and
//     looks at every id (they are few against the rows of dout, and in the L2
//     after the first look): a count of the ids below its rows is where its tokens
//     start in the sorted order, and counts of its own rows (by wavefront, each
//     walking a share of the tokens and listing those it finds) give every row's
//     start and every token its place.  One launch, where a radix sort takes
//     three for each digit.
//   embed_rows   A group of lanes owns a 16-byte chunk each of a row of dw: sums
//     its tokens' rows and writes it, zeros if it has none.  What hides the chain
//     from a row's start over its tokens to their rows is wavefronts, so they are
//     small: four rows in flight, not eight (63 us for 89 over 16384 tokens of
//     2048 and 32000 rows), a chunk a lane, not the whole row (51 for 71).  A row of more than kRun
//     tokens (a padding or end token, in the worst case all of them) is cut at
//     multiples of kRun positions of the sorted order, a group for each, into fp32
//     partials;
//   embed_fold   adds those of a row in order and writes it.
//
// Measured: 8192 rows of 4096 in bf16 looked up in 25 us (5.0 TB/s); their gradients of
// 16384 tokens of 2048 into 32000 rows 46 us, of them embed_rows 35 to 38 (5.4 TB/s),
// embed_index 10.
//
// Of few tokens and a small table the launches are most of the time: there
// embed_few does it all in one.  A workgroup owns a few rows of the table, or a part
// of their columns, looks at every id, a thread each, puts the tokens of its rows in
// order by counting, and its wavefronts sum and write the rows' pieces.
#include <algorithm>
#include <cmath>

#include "rowvec.h"
#include "workspace.h"

namespace mfx {
namespace embed {
namespace {

using namespace rowvec;

constexpr int kRun = 32;          // tokens that one group adds up
constexpr int kScanWaves = 16;    // of embed_index
constexpr int kScanRows = 480;    // table rows of one of its workgroups, at most (30 KB of counts)
constexpr int kScanList = 256;    // tokens that one of its wavefronts can list (32 KB in all)
constexpr int kFoldWaves = 4;
// embed_few: its tokens, a thread each; the table rows of one of its workgroups, at
// most; and the elements of dout and bytes of dw up to which it is taken.  Against the
// three launches, us: 257 x 512 tokens in 1000 rows 8.6 to 15.7, 64 x 4096 in 500 rows
// 7.9 to 11.9, 512 x 512 in 1000 rows 12.8 to 15.9; past the limits 257 x 4096 in 500
// rows 25 to 17, 64 x 512 in 32000 rows 16.4 to 14.9 (bf16, replayed from a graph).
constexpr int kFewTokens = 512;
constexpr int kFewRows = 512;
constexpr int64_t kFewElems = 1 << 18;
constexpr int64_t kFewBytes = 4 << 20;

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Elements a lane takes at a time: 16 bytes of the narrower type.
template <typename A, typename B>
constexpr int kVec = sizeof(A) == 4 && sizeof(B) == 4 ? 4 : 8;

// Group of LANES lanes of this launch (of fewer than 2^32 threads), uniform (a
// scalar) over a wavefront where the group is one.
template <int LANES>
__device__ __forceinline__ uint32_t group_id() {
  if constexpr (LANES == 64)
    return blockIdx.x * (kBlock / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  else
    return blockIdx.x * (kBlock / LANES) + threadIdx.x / LANES;
}

__device__ __forceinline__ int64_t load_id(const void* ids, int ids64, int64_t t) {
  return ids64 ? static_cast<const int64_t*>(ids)[t] : (int64_t)static_cast<const int32_t*>(ids)[t];
}

struct LookupArgs {
  const void* w;
  const void* ids;
  void* out;
  int64_t T, V, ws, os;
  int H, segs, ids64;
  float scale;
};

template <typename TI, typename TO, int LANES, int NV>
__global__ __launch_bounds__(kBlock) void embed_lookup(LookupArgs a) {
  constexpr int VEC = kVec<TI, TO>;
  const uint32_t g = group_id<LANES>(), row = g / (uint32_t)a.segs;
  const int64_t t = row;
  if (t >= a.T) return;
  const int col = (int)(g - row * a.segs) * (LANES * NV * VEC) + (int)(threadIdx.x % LANES) * VEC;
  const int64_t id = load_id(a.ids, a.ids64, t);
  const bool valid = id >= 0 && id < a.V;
  const TI* src = static_cast<const TI*>(a.w) + (valid ? id : 0) * a.ws;
  TO* dst = static_cast<TO*>(a.out) + t * a.os;
  float v[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    // (An id outside the table reads nothing.)
    load_run<TI, VEC>(src, col + i * LANES * VEC, valid ? a.H : 0, 0.f, v[i]);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[i][j] *= a.scale;
    store_run<TO, VEC>(dst, col + i * LANES * VEC, a.H, v[i]);
  }
}

// ---- the order of the tokens -----------------------------------------------------

struct IndexArgs {
  const void* ids;
  int32_t* order;
  int32_t* start;
  int64_t T, V;
  int ids64, rows;
};

// order[]: the tokens with an id in [0, V) by id, those of one id ascending;
// start[v]: where row v's begin, start[V] their number.
__global__ __launch_bounds__(kScanWaves * 64) void embed_index(IndexArgs a) {
  extern __shared__ int32_t count[];  // [wavefront][row]: tokens, then the next one's place
  __shared__ int32_t below_w[kScanWaves], scan_w[kScanWaves];
  __shared__ int2 list[kScanWaves][kScanList];  // (row, token)
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t T = a.T, V = a.V, v0 = (int64_t)blockIdx.x * a.rows;
  const int rows = a.rows, mine = (int)min((int64_t)rows, V - v0);
  const int bits = 32 - __clz((rows - 1) | 1);
  for (int i = tid; i < kScanWaves * rows; i += kScanWaves * 64) count[i] = 0;
  __syncthreads();

  // This wavefront's tokens.
  const int64_t per = (T + kScanWaves * 64 - 1) / (kScanWaves * 64) * 64;
  const int64_t t0 = min(T, wave * per), t1 = min(T, t0 + per);
  int32_t* const own = count + wave * rows;
  constexpr int U = 8;  // looks in flight
  // look(row or -1, or -2 below, token) for 64 tokens at a time.
  auto scan = [&](auto look) __attribute__((always_inline)) {
    for (int64_t t = t0; t < t1; t += 64 * U) {
      int64_t id[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t k = t + u * 64 + lane;
        id[u] = k < t1 ? load_id(a.ids, a.ids64, k) : -1;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t r = id[u] - v0;
        look(id[u] < 0 ? -1 : r < 0 ? -2 : r < mine ? (int)r : -1, (int32_t)(t + u * 64 + lane));
      }
    }
  };
  int32_t below = 0;
  int found = 0;  // of this wavefront
  scan([&](int r, int32_t t) __attribute__((always_inline)) {
    if (r == -2) ++below;
    const uint64_t in = __ballot(r >= 0);
    if (!in) return;
    if (r >= 0) {
      atomicAdd(own + r, 1);
      const int at = found + __popcll(in & ((1ull << lane) - 1));
      if (at < kScanList) list[wave][at] = make_int2(r, t);
    }
    found += __popcll(in);
  });
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) below += __shfl_xor(below, off, 64);
  if (lane == 0) below_w[wave] = below;
  __syncthreads();

  // Thread r: row r's tokens, their start, and each wavefront's.
  int32_t n = 0;
  if (tid < mine)
    for (int w = 0; w < kScanWaves; ++w) n += count[w * rows + tid];
  int32_t upto = n;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int32_t o = __shfl_up(upto, off, 64);
    if (lane >= off) upto += o;
  }
  if (lane == 63) scan_w[wave] = upto;
  __syncthreads();
  int32_t at = upto - n;
  for (int w = 0; w < kScanWaves; ++w) {
    at += below_w[w];
    if (w < wave) at += scan_w[w];
  }
  if (tid < mine) {
    a.start[v0 + tid] = at;
    if (v0 + tid == V - 1) a.start[V] = at + n;
    for (int w = 0; w < kScanWaves; ++w) {
      const int32_t c = count[w * rows + tid];
      count[w * rows + tid] = at;
      at += c;
    }
  }
  __syncthreads();

  // The lanes' tokens to their places, all 64 at once: the lanes with a lane's row
  // are found by the row's bits (one row at a time took 25 us where a workgroup
  // owned a fifth of 16384 tokens).
  auto place = [&](int r, int32_t t) __attribute__((always_inline)) {
    uint64_t same = __ballot(r >= 0);
    if (!same) return;
    for (int bit = 0; bit < bits; ++bit) {
      const uint64_t set = __ballot(r >= 0 && (r >> bit & 1));
      same &= r >> bit & 1 ? set : ~set;
    }
    if (r >= 0) {
      const int before = __popcll(same & ((1ull << lane) - 1)), all = __popcll(same);
      const int32_t to = own[r];
      a.order[to + before] = t;
      // (Every lane of the row has read its place: one instruction read them all.)
      if (before == all - 1) own[r] = to + all;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  };
  if (found <= kScanList) {
    for (int i = 0; i < found; i += 64) {
      const int2 x = i + lane < found ? list[wave][i + lane] : make_int2(-1, 0);
      place(x.x, x.y);
    }
  } else {
    scan(place);
  }
}

// ---- the sums --------------------------------------------------------------------

struct SumArgs {
  const void* dout;
  const void* ids;
  void* dw;
  const int32_t* order;
  const int32_t* start;
  float* part;       // [2 blocks][part_ld]: of the run at a block's first, and at its last position
  int64_t V, ds, gs, part_ld;
  int64_t blocks;    // of kRun positions (0: no row can have more tokens)
  int H, segs, ids64, add;  // segs: groups of a row
  float scale;
};

// Sum of the rows of dout at n <= kRun positions of the order, from s on; for a
// group of a wavefront their tokens are in its lanes.
template <typename T, int LANES, int VEC>
__device__ __forceinline__ void sum_rows(const SumArgs& a, int64_t s, int n, int32_t tokens, int col,
                                         float (&acc)[VEC]) {
  constexpr int U = 4;  // rows in flight
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
  const T* const dout = static_cast<const T*>(a.dout);
  for (int p = 0; p < n; p += U) {
    float v[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = p + u < n;
      const int32_t t = LANES == 64 ? __builtin_amdgcn_readlane(tokens, (p + u) & 63) : in ? a.order[s + p + u] : 0;
      load_run<T, VEC>(dout + (int64_t)t * a.ds, col, in ? a.H : 0, 0.f, v[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] += v[u][j];
  }
}

// (Past the caches: dw is written once and mostly larger than they are; 953 MB of
// f32 in 200 us for 270.)
template <typename TO, int VEC>
__device__ __forceinline__ void write_row(const SumArgs& a, int64_t v, int col, const float (&acc)[VEC]) {
  TO* const row = static_cast<TO*>(a.dw) + v * a.gs;
  float o[VEC];
  if (a.add) {
    load_run<TO, VEC>(row, col, a.H, 0.f, o);
#pragma unroll
    for (int j = 0; j < VEC; ++j) o[j] = fmaf(acc[j], a.scale, o[j]);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) o[j] = acc[j] * a.scale;
  }
  store_run<TO, VEC, true>(row, col, a.H, o);
}

template <typename TI, typename TO, int LANES>
__global__ __launch_bounds__(kBlock) void embed_rows(SumArgs a) {
  constexpr int VEC = kVec<TI, TO>;
  static_assert(kRun <= 64, "one load holds a run's tokens");
  const uint32_t g = group_id<LANES>(), which = g / (uint32_t)a.segs;
  int64_t task = which;
  const int lane = threadIdx.x % LANES;
  const int col = (int)(g - which * a.segs) * (LANES * VEC) + lane * VEC;
  float acc[VEC];
  int64_t s, e;
  // The blocks of long runs first: they take longest.
  const bool block = task < 2 * a.blocks;
  if (block) {
    const int64_t n = a.start[a.V], p0 = (task >> 1) * kRun, p1 = min(p0 + kRun, n);
    if (p0 >= n) return;
    const int64_t head = load_id(a.ids, a.ids64, a.order[p0]), tail = load_id(a.ids, a.ids64, a.order[p1 - 1]);
    if ((task & 1) && head == tail) return;
    const int64_t v = task & 1 ? tail : head;
    s = a.start[v], e = a.start[v + 1];
    if (e - s <= kRun) return;
    s = max(s, p0), e = min(e, p1);
  } else {
    task -= 2 * a.blocks;
    if (task >= a.V) return;
    s = a.start[task], e = a.start[task + 1];
    if (e - s > kRun || (a.add && s == e)) return;
  }
  const int n = (int)(e - s);
  const int32_t tokens = LANES == 64 && lane < n ? a.order[s + lane] : 0;
  sum_rows<TI, LANES, VEC>(a, s, n, tokens, col, acc);
  if (!block) {
    write_row<TO, VEC>(a, task, col, acc);
    return;
  }
  float* const to = a.part + task * a.part_ld + col;
#pragma unroll
  for (int j = 0; j < VEC; j += 4)
    if (col + j < a.H)  // (part_ld is H rounded up to whole chunks)
      *reinterpret_cast<f32x4*>(to + j) = f32x4{acc[j], acc[j + 1], acc[j + 2], acc[j + 3]};
}

// Workgroup (block, segment): the long run that starts in the block, if any.
template <typename TO>
__global__ __launch_bounds__(kFoldWaves * 64) void embed_fold(SumArgs a) {
  constexpr int VEC = 8, SEG = 64 * VEC;
  __shared__ float sums[kFoldWaves][SEG];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t segs = (a.H + SEG - 1) / SEG, b = blockIdx.x / segs;
  const int col = (int)(blockIdx.x - b * segs) * SEG + lane * VEC;
  const int64_t n = a.start[a.V], p0 = b * kRun, p1 = min(p0 + kRun, n);
  if (p0 >= n) return;
  const int64_t v = load_id(a.ids, a.ids64, a.order[p1 - 1]);
  const int64_t s = a.start[v], e = a.start[v + 1];
  if (s < p0 || e - s <= kRun) return;
  // Its partials: this block's, then the first-position ones of the blocks up to its end.
  const int64_t end = (e - 1) / kRun, parts = end - b + 1;
  const int64_t q0 = b + wave * parts / kFoldWaves, q1 = b + (wave + 1) * parts / kFoldWaves;
  float acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
  if (col < a.H) {
    constexpr int U = 8;
    for (int64_t q = q0; q < q1; q += U) {
      f32x4 x[U][2];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        // (Past the last: the last again, not added.)
        const int64_t k = min(q + u, q1 - 1), slot = 2 * k + (k == b && s > p0 ? 1 : 0);
        const f32x4* from = reinterpret_cast<const f32x4*>(a.part + slot * a.part_ld + col);
        x[u][0] = from[0];
        x[u][1] = from[1];
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (q + u < q1)
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[j] += x[u][j / 4][j % 4];
    }
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j) sums[wave][lane * VEC + j] = acc[j];
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int w = 1; w < kFoldWaves; ++w)
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] += sums[w][lane * VEC + j];
  if constexpr (sizeof(TO) == 4) {
    const float lo[4] = {acc[0], acc[1], acc[2], acc[3]}, hi[4] = {acc[4], acc[5], acc[6], acc[7]};
    write_row<TO, 4>(a, v, col, lo);
    write_row<TO, 4>(a, v, col + 4, hi);
  } else {
    write_row<TO, 8>(a, v, col, acc);
  }
}

// ---- few tokens in one launch --------------------------------------------------------

template <typename TI, typename TO>
__global__ __launch_bounds__(kFewTokens) void embed_few(SumArgs a, int tokens, int rows) {
  constexpr int VEC = kVec<TI, TO>, WAVES = kFewTokens / 64;
  __shared__ int found[kFewTokens];      // the rows of this workgroup's tokens, in the tokens' order
  __shared__ int16_t order[kFewTokens];  // the tokens by row
  __shared__ int count[kFewRows], start[kFewRows + 1], in_wave[WAVES];
  __shared__ float sums[WAVES][64 * VEC];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t v0 = (int64_t)blockIdx.x * rows;
  const int mine = (int)min((int64_t)rows, a.V - v0);
  const int seg0 = (int)((int64_t)a.segs * blockIdx.y / gridDim.y);
  const int segs = (int)((int64_t)a.segs * (blockIdx.y + 1) / gridDim.y) - seg0;
  const int64_t id = tid < tokens ? load_id(a.ids, a.ids64, tid) : -1;
  const bool in = id >= v0 && id < v0 + mine;
  const uint64_t hits = __ballot(in);
  if (lane == 0) in_wave[wave] = (int)__popcll(hits);
  if (tid < rows) count[tid] = 0;
  __syncthreads();
  int at = (int)__popcll(hits & ((1ull << lane) - 1));
#pragma unroll
  for (int w = 0; w < WAVES; ++w)
    if (w < wave) at += in_wave[w];
  const int r = in ? (int)(id - v0) : 0;
  if (in) {
    found[at] = r;
    atomicAdd(count + r, 1);
  }
  __syncthreads();
  static_assert(kFewRows <= kFewTokens, "a thread for each row");
  if (tid < mine) {
    int s = 0;
    for (int k = 0; k < tid; ++k) s += count[k];
    start[tid] = s;
    // (The last row's end too: a workgroup of kFewRows rows has no thread behind its last.)
    if (tid == mine - 1) start[mine] = s + count[tid];
  }
  __syncthreads();
  if (in) {
    int place = start[r];
    for (int k = 0; k < at; ++k) place += found[k] == r;
    order[place] = (int16_t)tid;
  }
  __syncthreads();

  const TI* const dout = static_cast<const TI*>(a.dout);
  // Sum of the tokens [s, e) of the order.
  auto sum = [&](int s, int e, int col, float (&acc)[VEC]) __attribute__((always_inline)) {
    constexpr int U = 8;  // rows in flight
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
    for (int p = s; p < e; p += U) {
      float v[U][VEC];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool one = p + u < e;
        const int t = one ? __builtin_amdgcn_readfirstlane(order[p + u]) : 0;
        load_run<TI, VEC>(dout + (int64_t)t * a.ds, col, one ? a.H : 0, 0.f, v[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] += v[u][j];
    }
  };
  float acc[VEC];
  // A wavefront to each piece of a row of few tokens ...
  for (int task = wave; task < mine * segs; task += WAVES) {
    const int row = task / segs, col = (seg0 + task - row * segs) * (64 * VEC) + lane * VEC;
    const int s = start[row], e = start[row + 1];
    if (e - s > kRun || (a.add && s == e)) continue;
    sum(s, e, col, acc);
    write_row<TO, VEC>(a, v0 + row, col, acc);
  }
  // ... and all of them a share of the tokens of a row of more.
  for (int row = 0; row < mine; ++row) {
    const int s = start[row], n = start[row + 1] - s;
    if (n <= kRun) continue;
    for (int seg = 0; seg < segs; ++seg) {
      const int col = (seg0 + seg) * (64 * VEC) + lane * VEC;
      sum(s + n * wave / WAVES, s + n * (wave + 1) / WAVES, col, acc);
#pragma unroll
      for (int j = 0; j < VEC; ++j) sums[wave][lane * VEC + j] = acc[j];
      __syncthreads();
      if (wave == 0) {
#pragma unroll
        for (int w = 1; w < WAVES; ++w)
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[j] += sums[w][lane * VEC + j];
        write_row<TO, VEC>(a, v0 + row, col, acc);
      }
      __syncthreads();
    }
  }
}

// ---- host ------------------------------------------------------------------------

bool float_dtype(int dt) { return dt == MFX_F32 || dt == MFX_BF16 || dt == MFX_F16; }

// Lanes of a group and 16-byte chunks a lane takes: 16 lanes for rows that a
// wavefront would leave mostly idle; four chunks a lane where that still makes
// eight wavefronts a CU (a launch of fewer is bound by latency and wants as many as
// it can have).
struct Split {
  int lanes, nv, segs;
};
Split split(int64_t rows, int64_t H, int vec, int most) {
  Split s{H <= 16 * vec ? 16 : 64, 1, 1};
  if (s.lanes == 64) {
    const int64_t chunks = ceil_div(H, 64 * vec);
    while (s.nv * 2 <= most && s.nv < chunks && rows * ceil_div(chunks, s.nv * 2) >= 8LL * device_cu_count()) s.nv *= 2;
  }
  s.segs = (int)ceil_div(H, (int64_t)s.lanes * vec * s.nv);
  return s;
}

int vec_of(int a, int b) { return a == MFX_F32 && b == MFX_F32 ? 4 : 8; }

int check_common(int64_t T, int64_t H, int64_t V, int dtype, int other, int ids_dtype, float scale, const char* what) {
  const int64_t lim = 0x7fffffffLL - 4096;
  if (T < 0 || H <= 0 || V <= 0) return fail(MFX_E_INVALID, "T must be >= 0, H and V positive");
  if (!float_dtype(dtype) || !float_dtype(other))
    return fail(MFX_E_UNSUPPORTED, std::string("dtype and ") + what + " must be f32, bf16 or f16");
  if (ids_dtype != MFX_I32 && ids_dtype != MFX_I64) return fail(MFX_E_UNSUPPORTED, "ids dtype must be i32 or i64");
  if (!std::isfinite(scale)) return fail(MFX_E_INVALID, "scale must be finite");
  if (T > lim || V > lim || H > lim) return fail(MFX_E_UNSUPPORTED, "T, H or V too large");
  return MFX_OK;
}

// (Rows that are only read may overlap: a gradient broadcast over the tokens.)
int check_rows(const void* p, int64_t stride, int64_t rows, int64_t H, int dtype, const char* what, bool written) {
  if (!p) return fail(MFX_E_INVALID, std::string(what) + " must be non-null");
  if ((uintptr_t)p % dtype_size(dtype)) return fail(MFX_E_INVALID, std::string(what) + " must be aligned to its type");
  if (rows > 1 && stride < (written ? H : 0))
    return fail(MFX_E_INVALID, std::string(what) + (written ? ": row stride must be >= H" : ": row stride must be >= 0"));
  return MFX_OK;
}

int check_ids(const void* ids, int dtype) {
  if (!ids) return fail(MFX_E_INVALID, "ids must be non-null");
  if ((uintptr_t)ids % (dtype == MFX_I64 ? 8 : 4)) return fail(MFX_E_INVALID, "ids must be aligned to their type");
  return MFX_OK;
}

struct FwdPlan {
  Split sp;
  int64_t grid;
};
int plan_fwd(const mfx_embedding_args* a, FwdPlan& pl) {
  if (!a) return fail(MFX_E_INVALID, "null args");
  if (int rc = check_common(a->T, a->H, a->V, a->dtype, a->out_dtype, a->ids_dtype, a->scale, "out_dtype")) return rc;
  if (a->T == 0) return MFX_OK;
  if (int rc = check_ids(a->ids, a->ids_dtype)) return rc;
  if (int rc = check_rows(a->w, a->w_stride, a->V, a->H, a->dtype, "w", false)) return rc;
  if (int rc = check_rows(a->out, a->out_stride, a->T, a->H, a->out_dtype, "out", true)) return rc;
  pl.sp = split(a->T, a->H, vec_of(a->dtype, a->out_dtype), 4);
  pl.grid = ceil_div(a->T * pl.sp.segs, kBlock / pl.sp.lanes);
  if (!launch_fits(pl.grid, kBlock)) return fail(MFX_E_UNSUPPORTED, "problem too large for one launch");
  return MFX_OK;
}

struct BwdPlan {
  bool few;  // embed_few: `scans` by `grid` workgroups of `rows` rows and a part of the columns, no workspace
  int lanes, segs;
  int64_t blocks, grid, fold, part_ld;
  int rows;
  int64_t scans;
  size_t order_bytes, start_bytes, part_bytes, total;
};
int plan_bwd(const mfx_embedding_bwd_args* a, BwdPlan& pl) {
  if (!a) return fail(MFX_E_INVALID, "null args");
  if (int rc = check_common(a->T, a->H, a->V, a->dtype, a->dw_dtype, a->ids_dtype, a->scale, "dw_dtype")) return rc;
  if (int rc = check_rows(a->dw, a->dw_stride, a->V, a->H, a->dw_dtype, "dw", true)) return rc;
  if (a->T > 0) {
    if (int rc = check_ids(a->ids, a->ids_dtype)) return rc;
    if (int rc = check_rows(a->dout, a->dout_stride, a->T, a->H, a->dtype, "dout", false)) return rc;
  }
  const int vec = vec_of(a->dtype, a->dw_dtype);
  pl.few = a->T <= kFewTokens && a->T * a->H <= kFewElems &&
           a->V * a->H * dtype_size(a->dw_dtype) <= kFewBytes;
  if (pl.few) {
    // Two workgroups a CU at most.
    pl.segs = (int)ceil_div(a->H, 64 * vec);
    pl.rows = (int)std::min<int64_t>(kFewRows, ceil_div(a->V, 2 * device_cu_count()));
    pl.scans = ceil_div(a->V, pl.rows);
    pl.grid = std::min<int64_t>(pl.segs, std::max<int64_t>(1, 2 * device_cu_count() / pl.scans));
    pl.order_bytes = pl.start_bytes = pl.part_bytes = pl.total = 0;
    return MFX_OK;
  }
  pl.lanes = a->H <= 16 * vec ? 16 : 64;
  pl.segs = (int)ceil_div(a->H, pl.lanes * vec);
  pl.blocks = a->T > kRun ? ceil_div(a->T, kRun) : 0;
  pl.grid = ceil_div((2 * pl.blocks + a->V) * pl.segs, kBlock / pl.lanes);
  pl.fold = pl.blocks * ceil_div(a->H, 512);
  // A workgroup of the index for each CU, of at most 480 rows (a thread each).
  pl.rows = (int)std::min<int64_t>(kScanRows, ceil_div(a->V, device_cu_count()));
  pl.scans = ceil_div(a->V, pl.rows);
  if (!launch_fits(pl.grid, kBlock) || !launch_fits(pl.fold, kFoldWaves * 64) ||
      !launch_fits(pl.scans, kScanWaves * 64))
    return fail(MFX_E_UNSUPPORTED, "problem too large for one launch");
  pl.part_ld = ceil_div(a->H, 8) * 8;
  pl.order_bytes = align256((size_t)a->T * 4);
  pl.start_bytes = align256(((size_t)a->V + 1) * 4);
  pl.part_bytes = (size_t)pl.blocks * 2 * pl.part_ld * 4;
  pl.total = pl.order_bytes + pl.start_bytes + pl.part_bytes;
  return MFX_OK;
}

template <typename TI, typename TO>
void launch_lookup(const LookupArgs& p, const FwdPlan& pl, hipStream_t s) {
  const dim3 grid((unsigned)pl.grid), block(kBlock);
  if (pl.sp.lanes == 16) hipLaunchKernelGGL((embed_lookup<TI, TO, 16, 1>), grid, block, 0, s, p);
  else if (pl.sp.nv == 1) hipLaunchKernelGGL((embed_lookup<TI, TO, 64, 1>), grid, block, 0, s, p);
  else if (pl.sp.nv == 2) hipLaunchKernelGGL((embed_lookup<TI, TO, 64, 2>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((embed_lookup<TI, TO, 64, 4>), grid, block, 0, s, p);
}

template <typename TI, typename TO>
void launch_rows(const SumArgs& p, const BwdPlan& pl, int64_t T, hipStream_t s) {
  if (pl.few) {
    hipLaunchKernelGGL((embed_few<TI, TO>), dim3((unsigned)pl.scans, (unsigned)pl.grid),
                       dim3(kFewTokens), 0, s, p, (int)T, pl.rows);
    return;
  }
  const dim3 grid((unsigned)pl.grid), block(kBlock);
  if (pl.lanes == 16) hipLaunchKernelGGL((embed_rows<TI, TO, 16>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((embed_rows<TI, TO, 64>), grid, block, 0, s, p);
}

// f(TI{}, TO{}) for a pair of element types.
template <class F>
void with_types(int in, int out, F f) {
  auto second = [&](auto t) {
    if (out == MFX_F32) f(t, float{});
    else if (out == MFX_BF16) f(t, bf16{});
    else f(t, _Float16{});
  };
  if (in == MFX_F32) second(float{});
  else if (in == MFX_BF16) second(bf16{});
  else second(_Float16{});
}

}  // namespace
}  // namespace embed
}  // namespace mfx

extern "C" {

int mfx_embedding(const mfx_embedding_args* args, void* stream) {
  using namespace mfx;
  using namespace mfx::embed;
  FwdPlan pl;
  if (int rc = plan_fwd(args, pl)) return rc;
  const mfx_embedding_args& a = *args;
  if (a.T == 0) return MFX_OK;
  const LookupArgs p{a.w, a.ids, a.out, a.T, a.V, a.w_stride, a.out_stride, (int)a.H, pl.sp.segs,
                     a.ids_dtype == MFX_I64, a.scale};
  with_types(a.dtype, a.out_dtype, [&](auto ti, auto to) {
    launch_lookup<decltype(ti), decltype(to)>(p, pl, static_cast<hipStream_t>(stream));
  });
  return launch_status("embed_lookup");
}

size_t mfx_embedding_bwd_workspace_size(const mfx_embedding_bwd_args* args) {
  mfx::embed::BwdPlan pl;
  return mfx::embed::plan_bwd(args, pl) == MFX_OK ? pl.total : 0;
}

int mfx_embedding_bwd(const mfx_embedding_bwd_args* args, void* stream) {
  using namespace mfx;
  using namespace mfx::embed;
  BwdPlan pl;
  if (int rc = plan_bwd(args, pl)) return rc;
  const mfx_embedding_bwd_args& a = *args;
  if (a.T == 0 && a.accumulate) return MFX_OK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* ws = nullptr;
  if (int rc = take_workspace(a.workspace, a.workspace_bytes, pl.total, "mfx_embedding_bwd_workspace_size", s, &ws))
    return rc;
  int32_t* const order = reinterpret_cast<int32_t*>(ws);
  int32_t* const start = reinterpret_cast<int32_t*>(ws + pl.order_bytes);
  const int ids64 = a.ids_dtype == MFX_I64;
  if (!pl.few) {
    const IndexArgs x{a.ids, order, start, a.T, a.V, ids64, pl.rows};
    hipLaunchKernelGGL(embed_index, dim3((unsigned)pl.scans), dim3(kScanWaves * 64), (size_t)kScanWaves * pl.rows * 4, s,
                       x);
    if (int rc = launch_status("embed_index")) return rc;
  }
  const SumArgs p{a.dout, a.ids, a.dw, order, start, reinterpret_cast<float*>(ws + pl.order_bytes + pl.start_bytes),
                  a.V, a.dout_stride, a.dw_stride, pl.part_ld, pl.blocks, (int)a.H, pl.segs, ids64,
                  a.accumulate != 0, a.scale};
  with_types(a.dtype, a.dw_dtype, [&](auto ti, auto to) { launch_rows<decltype(ti), decltype(to)>(p, pl, a.T, s); });
  if (int rc = launch_status(pl.few ? "embed_few" : "embed_rows")) return rc;
  if (pl.few || !pl.blocks) return MFX_OK;
  const dim3 grid((unsigned)pl.fold), block(kFoldWaves * 64);
  if (a.dw_dtype == MFX_F32) hipLaunchKernelGGL((embed_fold<float>), grid, block, 0, s, p);
  else if (a.dw_dtype == MFX_BF16) hipLaunchKernelGGL((embed_fold<bf16>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((embed_fold<_Float16>), grid, block, 0, s, p);
  return launch_status("embed_fold");
}

}  // extern "C"

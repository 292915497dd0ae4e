// Packed sequences: where a workgroup of an attention kernel finds its rows.
//
// A packed batch is T tokens, sequence s of them from off[s] up to off[s + 1],
// the offsets in device memory.  The host knows neither the lengths nor the
// number of row blocks, only a bound: a sequence of n rows is at most
// n / BM + 1 blocks, so T / BM slots per head and one for each sequence that
// can hold a token cover all.
// Each workgroup finds its own (sequence, block) from its slot number, with
// no launch before it, and slots without a block leave at once.
//
// Order.  Under a causal mask block b of a sequence walks b + 1 blocks of
// keys (a block of keys, the blocks of queries behind it), so blocks are handed
// out by that number, longest first, over all sequences: workgroups start in
// slot order, and a long block started last would run alone.  With nb(s)
// blocks in sequence s, above(w) = sum_s max(nb(s) - w, 0) blocks have work
// past w; slot r belongs to the w with above(w + 1) <= r < above(w), found by
// bisection, each lane holding the nb of its sequences, and to the
// (r - above(w + 1))-th sequence of more than w blocks.  That takes a bisection
// step of a few vector operations and one sum over the lanes (about 80
// cycles), some 8 steps.  Past kLaneSeqs sequences a lane's share no longer
// fits registers, and slots go to sequences in order: sequence s owns the slots
// from (off[s] - off[0]) / BM + s, which are enough for it and need no count
// of the blocks before (empty sequences own one too).  What the order is worth
// there is less than what it costs to find: one sequence of 4096 tokens and 511 of
// 8, 32 heads on 8 of 128, forward 355 us and backward 1033, with 512 of 8 295
// and 941; one of 8192 and 500 of 4 707 and 2392, 520 of 4 653 and 2320.
//
// Offsets are taken as they come: each is clamped to 0 .. T and a sequence that
// would end before it starts is empty, so no offsets lead outside the tensors.
#pragma once

#include <type_traits>

#include "packed_index.h"
#include "sdpa_common.h"

namespace mfx {

constexpr int kCus = 256;  // of the whole MI355X (a partition with fewer is only shared out finer than it needs)
constexpr int kLaneSeqs = 8;  // sequences a lane holds: 512 in all
constexpr int kPartTiles = 8;  // blocks of so many tiles have one share

struct PackedBlock {
  int start, len;  // the sequence's first token and its length
  int work;        // key blocks behind this one, 0 .. nb - 1 (see above)
  int nb;          // its blocks
};

// Sum over the wavefront's 64 lanes, in every lane.
__device__ __forceinline__ int wave_sum(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // from 1, 2, 4, 8 lanes below, within 16
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // lane 15's and 47's into the 16 above
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // lane 31's into the upper half
  return __builtin_amdgcn_readlane(v, 63);
}

__device__ __forceinline__ void packed_bounds(const int32_t* off, int total, int s, int& start, int& len) {
  start = min(max(off[s], 0), total);
  len = max(min(off[s + 1], total) - start, 0);
}

// First slot of sequence s, which starts at `at`, when slots go in order.
template <int BM>
__device__ __forceinline__ int64_t packed_slot(int at, int first, int s) {
  const int64_t d = (int64_t)at - first;
  return (d > 0 ? d : 0) / BM + s;
}

// Slot `r`'s block of BM rows; false: it has none.  Uniform over the
// wavefront (every lane active).
template <int BM>
__device__ __forceinline__ bool packed_block(const int32_t* off, int n, int total, int r, PackedBlock& out) {
  const int lane = threadIdx.x & 63;
  int seq, work;
  if (n <= 64 * kLaneSeqs) {
    int nb[kLaneSeqs];
#pragma unroll
    for (int c = 0; c < kLaneSeqs; ++c) {
      nb[c] = 0;
      if (c * 64 < n) {
        int a, len = 0;
        if (c * 64 + lane < n) packed_bounds(off, total, c * 64 + lane, a, len);
        nb[c] = (len + BM - 1) / BM;
      }
    }
    auto above = [&](int w) {
      int v = 0;
#pragma unroll
      for (int c = 0; c < kLaneSeqs; ++c)
        if (c * 64 < n) v += max(nb[c] - w, 0);
      return wave_sum(v);
    };
    if (above(0) <= r) return false;
    int lo = 0, hi = (total + BM - 1) / BM;  // above(lo) > r >= above(hi)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (above(mid) > r) lo = mid;
      else hi = mid;
    }
    work = lo;
    int j = r - above(lo + 1);
    seq = 0;
    bool found = false;
#pragma unroll
    for (int c = 0; c < kLaneSeqs; ++c) {
      if (c * 64 < n && !found) {
        const uint64_t m = __ballot(nb[c] > lo);
        const int cnt = __popcll(m);
        if (j < cnt) {
          const bool mine = (m >> lane & 1) && __popcll(m & ((1ull << lane) - 1)) == j;
          seq = c * 64 + __builtin_ctzll(__ballot(mine));
          found = true;
        }
        j -= cnt;
      }
    }
    packed_bounds(off, total, __builtin_amdgcn_readfirstlane(seq), out.start, out.len);
    out.nb = (out.len + BM - 1) / BM;
  } else {
    // The last sequence whose first slot is at or before r, 64 at a time.
    const int first = off[0];
    int lo = 0, hi = n;
    while (hi - lo > 1) {
      const int step = (hi - lo + 63) / 64, s = lo + lane * step;
      const bool at = s < hi && packed_slot<BM>(off[min(s, n)], first, s) <= r;
      const int cnt = max(__popcll(__ballot(at)), 1);
      lo += (cnt - 1) * step;
      hi = min(hi, lo + step);
    }
    seq = __builtin_amdgcn_readfirstlane(lo);
    packed_bounds(off, total, seq, out.start, out.len);
    const int64_t b = r - packed_slot<BM>(off[seq], first, seq);
    out.nb = (out.len + BM - 1) / BM;
    if (b < 0 || b >= out.nb) return false;
    work = out.nb - 1 - (int)b;
  }
  out.start = __builtin_amdgcn_readfirstlane(out.start);
  out.len = __builtin_amdgcn_readfirstlane(out.len);
  out.nb = __builtin_amdgcn_readfirstlane(out.nb);
  out.work = __builtin_amdgcn_readfirstlane(work);
  return true;
}

// Blocks in shares.  Under a causal mask a block with work w walks
// `tiles` (w + 1) tiles; one that walks more than `most` is shared
// by as many workgroups as bring each to `most` or less, at most sh.parts.
// `most` is sh.quarters quarters of what each of `room` workgroups at a time
// gets of all tiles of `heads` heads, or `least` if that is more.  Blocks are
// handed out by w, longest first, so those of most shares come first: with
// n(k) blocks of k shares or more, whose w is (k - 1) most / tiles or more,
// slot r falls to block and share by a walk over k, and no workgroup is
// without work before the last.  (Every other workgroup leaving at once leaves
// half the shader engines without work: a batch of 8192 tokens took 1.4 times
// as long.)
struct PackedShare {
  int block, part, parts;
};
template <int BM, class Params>
__device__ __forceinline__ PackedShare packed_share(const Params& p, const PackedShares& sh, int heads, int room,
                                                    int tiles, int least, int r) {
  int nb[kLaneSeqs];
  int work = 0;
#pragma unroll
  for (int c = 0; c < kLaneSeqs; ++c) {
    nb[c] = 0;
    if (c * 64 < p.num_seqs) {
      int a, len = 0;
      const int s = c * 64 + (threadIdx.x & 63);
      if (s < p.num_seqs) packed_bounds(p.seq_off, p.total, s, a, len);
      nb[c] = (len + BM - 1) / BM;
      work += nb[c] * (nb[c] + 1) / 2;
    }
  }
  const int64_t all = (int64_t)wave_sum(work) * tiles * heads * sh.quarters;
  const int most = max((int)min((all + 4 * room - 1) / (4 * room), (int64_t)1 << 27), least);
  PackedShare out{0, 0, 1};
  int before = 0, base = 0;
  for (int k = sh.parts; k > 1; --k) {
    const int w = (k - 1) * most / tiles;
    int v = 0;
#pragma unroll
    for (int c = 0; c < kLaneSeqs; ++c)
      if (c * 64 < p.num_seqs) v += max(nb[c] - w, 0);
    const int n = wave_sum(v) - before;  // of exactly k (the first: at least)
    if (r < base + n * k) {
      out.block = before + (r - base) / k;
      out.part = (r - base) % k;
      out.parts = k;
      return out;
    }
    base += n * k;
    before += n;
  }
  out.block = before + r - base;
  return out;
}

// The sequence that token t lies in; false: none.
__device__ __forceinline__ bool packed_seq(const int32_t* off, int n, int total, int t, int& start, int& len) {
  int lo = 0, hi = n;  // the last s with off[s] <= t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (off[mid] <= t) lo = mid;
    else hi = mid;
  }
  packed_bounds(off, total, lo, start, len);
  return t >= start && t < start + len;
}

// The tokens in no sequence: those before `first` and from `last` on.  Their
// offsets are loaded where this is made, used where rows are zeroed: a kernel
// makes it before it looks for its block, whose loads then travel beside these
// (a call of 325 tokens: 0.2 us more with the loads one behind the other).
struct PackedRest {
  int first, last, total;
  __device__ __forceinline__ PackedRest(const int32_t* off, int n, int t) : first(off[0]), last(off[n]), total(t) {}
};

// The last workgroups of a grid zero those rows: their blocks are the shortest,
// or they have none, and the others need not wait for what to do (4 us of a
// 500 us backward, in which every workgroup asked).
constexpr uint32_t kRestGroups = 2 * kCus;
__device__ __forceinline__ bool packed_rest_here() { return blockIdx.x + kRestGroups >= gridDim.x; }

// Zeros in those rows of a [heads, total, D] tensor of whole, aligned 16-byte
// chunks, shared out over these workgroups of NT threads; up to 64 chunks a row.
// (The products and sums that take the tensor next go over every row.)
template <int SIZE, int NT>
__device__ __forceinline__ void packed_zero_rest(const PackedRest& rest, void* out, const int64_t (&st)[4], int heads,
                                                 int D) {
  const int total = rest.total, first = min(max(rest.first, 0), total), last = max(min(rest.last, total), first);
  // (Fewer than 2^31 rows, and 2^32 threads in the grid: checked on the host.)
  const uint32_t rows = (uint32_t)(first + total - last) * (uint32_t)heads;
  if (rows == 0) return;
  const uint32_t groups = min((uint32_t)gridDim.x, kRestGroups), group = blockIdx.x + groups - gridDim.x;
  const uint32_t chunks = D * SIZE / 16, per = NT / chunks;  // of a row; rows a workgroup takes at a time
  const uint32_t mine = threadIdx.x / chunks, chunk = threadIdx.x - mine * chunks;
  if (mine >= per) return;
  for (uint32_t r = group * per + mine; r < rows; r += groups * per) {
    int t = (int)(r / (uint32_t)heads);
    const int h = (int)(r - (uint32_t)t * (uint32_t)heads);
    if (t >= first) t += last - first;
    char* const row = static_cast<char*>(out) + (h * st[1] + t * st[2]) * SIZE;
    *reinterpret_cast<u32x4*>(row + chunk * 16) = u32x4{0, 0, 0, 0};
  }
}

// Zeros in one row, by a wavefront.
template <typename T>
__device__ __forceinline__ void packed_zero_row(void* out, const int64_t (&st)[4], int h, int t, int D) {
  T* const row = static_cast<T*>(out) + h * st[1] + t * st[2];
  for (int d = threadIdx.x & 63; d < D; d += 64) row[d] = static_cast<T>(0.f);
}

// Slots per head of a packed call (host): blocks of BM rows at most, and past
// 64 kLaneSeqs sequences a slot for every empty one too.
inline int64_t packed_slots(int64_t total, int64_t n, int BM) {
  return total / BM + (n <= 64 * kLaneSeqs && total < n ? total : n);
}

// (head, slot) of a workgroup.  Workgroups are dealt to the 8 XCDs in turn;
// with heads divisible by 8 each XCD takes a run of neighbouring heads, which
// share K and V under grouped queries, four at a time side by side.
__device__ __forceinline__ void packed_head(int id, int heads, int slots, int& head, int& slot) {
  if ((heads & 7) == 0) {
    const int per = heads >> 3, hg = (per & 3) == 0 ? 4 : (per & 1) == 0 ? 2 : 1;
    const int i = id >> 3, r = i % (hg * slots);
    head = (id & 7) * per + i / (hg * slots) * hg + r % hg;
    slot = r / hg;
  } else {
    head = id % heads;
    slot = id / heads;
  }
}

// Points the params at the rows of one sequence (batch 1): SIZE-byte elements.
template <int SIZE>
__device__ __forceinline__ void packed_shift(SdpaParams& p, int start, int len) {
  auto at = [&](auto*& ptr, int64_t stride) {
    ptr = reinterpret_cast<std::remove_reference_t<decltype(ptr)>>(
        reinterpret_cast<uintptr_t>(ptr) + (int64_t)start * stride * SIZE);
  };
  at(p.q, p.qs[2]);
  at(p.k, p.ks[2]);
  at(p.v, p.vs[2]);
  at(p.out, p.os[2]);
  if (p.lse) p.lse += start;
  p.Tq = p.Tk = len;
}
template <int SIZE>
__device__ __forceinline__ void packed_shift(SdpaBwdParams& p, int start, int len) {
  auto at = [&](auto*& ptr, int64_t stride) {
    ptr = reinterpret_cast<std::remove_reference_t<decltype(ptr)>>(
        reinterpret_cast<uintptr_t>(ptr) + (int64_t)start * stride * SIZE);
  };
  at(p.q, p.qs[2]);
  at(p.k, p.ks[2]);
  at(p.v, p.vs[2]);
  at(p.o, p.os[2]);
  at(p.dout, p.dos[2]);
  at(p.dq, p.dqs[2]);
  at(p.dk, p.dks[2]);
  at(p.dv, p.dvs[2]);
  p.lse += start;
  p.delta += start;
  p.Tq = p.Tk = len;
}

// Rows of lse and delta from one head to the next.
template <bool PACKED, class Params>
__device__ __forceinline__ int row_pitch(const Params& p) {
  if constexpr (PACKED) return p.total;
  else return p.Tq;
}

// The kernels' packed instances (batch 1, Tq = Tk = the tokens, no mask).
int launch_packed_flash16(const SdpaParams& p, hipStream_t s);
int launch_packed_f32(const SdpaParams& p, hipStream_t s);
int launch_packed_generic(const SdpaParams& p, hipStream_t s);
int launch_packed_bwd_mfma(const SdpaBwdParams& p, hipStream_t s);
constexpr int kBwdBlock = 128;  // keys (or queries) a workgroup of it owns
int launch_packed_bwd_f32(const SdpaBwdParams& p, hipStream_t s);
int launch_packed_bwd_generic(const SdpaBwdParams& p, hipStream_t s);
// Copies a [1, H, total, D] tensor into rows of dp features (or back, rows in
// a sequence only, and with `zero` zeros in the others).
int packed_pad_rows(const void* src, void* dst, const SdpaBwdParams& p, int H, int dp, const int64_t* st, bool unpad,
                    bool zero, hipStream_t s);

}  // namespace mfx

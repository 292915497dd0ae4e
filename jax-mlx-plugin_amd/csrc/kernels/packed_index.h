// Index arithmetic of the packed attention kernels (sdpa_packed.h) that large
// calls can take past 31 bits.  Header-only and free of HIP so host tests can
// check it at sizes that no test runs.
#pragma once

#include <cstdint>

namespace mfx {

// The share count that thread `tid` of workgroup `id` (of `threads`) clears,
// of `counts` in all; -1: none.  Empty sequences past 512 own a slot for every
// head, so a call of few tokens may have 2^23 workgroups and more: id *
// threads does not fit 31 bits then.
constexpr int64_t packed_cleared(uint32_t id, int tid, int threads, int64_t counts) {
  const int64_t i = (int64_t)id * threads + tid;
  return i < counts ? i : -1;
}

// Whether any block of a packed call can be worked on in shares
// (packed_share).  Block m of a sequence, counted from 1 by its keys, walks
// tiles * m tiles and is shared if they are more than `most`, which is `least` or
// more and quarters / (4 room) of the tiles of `heads` heads or more.  A
// sequence with a block m has m (m + 1) / 2 blocks' worth of `tiles` in all, so
// heads * quarters * (m + 1) < 8 room has to hold, and the first m of more than
// `least` tiles has to exist in `total` tokens of BM a block.
constexpr bool packed_shares_possible(int64_t total, int BM, int64_t heads, int quarters, int room, int64_t tiles,
                                      int least) {
  const int64_t m = least / tiles + 1;
  return m <= (total + BM - 1) / BM && heads * quarters * (m + 1) < 8 * (int64_t)room;
}

}  // namespace mfx

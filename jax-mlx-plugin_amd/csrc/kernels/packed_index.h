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

}  // namespace mfx

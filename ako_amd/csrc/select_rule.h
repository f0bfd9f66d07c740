// How many token rows a launch over blocks of a paged cache takes, so that its work-items stay below 2^32. Plain C++:
// paged_select.hip launches by it, and a CPU test goes through its sizes.
#pragma once

#include <stdint.h>

#include <algorithm>

namespace ako {

// Work-items of a launch, at most; a call of more rows is launched in slices.
constexpr int64_t kSliceItems = int64_t(1) << 30;
// Workgroups of `threads` work-items in a slice.
constexpr int64_t slice_groups(int threads) { return kSliceItems / threads; }

// Work-items of a workgroup that scores and chooses for a tile of token rows. Single rows are few workgroups, each of a whole row: 16
// wavefronts to have more of it in flight, where the registers allow.
constexpr int tile_threads(int head_dim, bool one) { return one && head_dim <= 128 ? 1024 : 512; }

// Token rows of a slice of such workgroups, one for each tile and key head: whole tiles, one at least (key heads
// are fewer than 2^15).
inline int64_t tile_slice(int64_t head_dim, int64_t tile, int64_t kv_heads) {
  return std::max<int64_t>(1, slice_groups(tile_threads(static_cast<int>(head_dim), tile == 1)) / kv_heads) * tile;
}

}  // namespace ako

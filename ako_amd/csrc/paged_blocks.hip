// Attention of a step's tokens over the blocks of a paged cache that are listed for each of
// them, on gfx950: attn_rows with BLOCKS (paged_rows.h), and how a call is cut up.
//
// 16 tokens of 4096 keys of 8 key heads in 8 bits, 138 MB: 40 us with the join, 3.5 TB/s. 2048 tokens, each with 1024 keys of
// its own choosing: 420 us, 5.3 GB from L2 at 12.6 TB/s; four tokens share a tile, but hardly any blocks.

#include "paged_rows.h"

namespace ako {
namespace {

// Known from what the host knows of a call, so that the workspace can be sized before it.
struct Plan {
  bool once;           // (nearly) every key is read by one workgroup only
  int64_t row_tiles;   // of 16 rows for one key head, at most
  int parts;           // of every row tile's keys
  int64_t slots;       // row tiles of parts, of all key heads
};

Plan plan(const PagedAttentionArgs& a) {
  const int64_t group = a.q_heads / a.c.kv_heads;
  Plan p{};
  const int64_t rows = a.c.n_seqs > 0 ? ceil_div(a.c.tokens * group, a.c.n_seqs) : 1;
  p.row_tiles = a.c.cu ? a.c.tokens * group / 16 + a.c.n_seqs + 1 : a.c.n_seqs * ceil_div(rows, 16);
  p.once = rows <= 16;
  // Two workgroups to a CU, in one round, as each finds its blocks anew: 16 tokens of 4096 keys, 8 key heads, in 8
  // bits, 256 / 512 / 1024 workgroups 51.7 / 40.5 / 47.2 us. Parts of 128 keys, a tile for each
  // wavefront: one token of 1024 keys in parts of 64 / 128 / 256 12.2 / 12.0 / 13.6.
  const int64_t items = a.tuned_items > 0 ? a.tuned_items : 512, least = a.tuned_min_keys > 0 ? a.tuned_min_keys : 128;
  const int64_t keys = std::min(a.c.table_width, a.block_count) * a.c.page_size;
  const int64_t parts = std::min(items / std::max<int64_t>(1, p.row_tiles * a.c.kv_heads), keys / least);
  p.parts = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kMaxParts, parts)));
  p.slots = p.parts > 1 ? p.row_tiles * p.parts * a.c.kv_heads : 0;
  return p;
}

template <typename T, bool MX, int DP>
hipError_t run(const PagedAttentionArgs& a, hipStream_t stream) {
  const Plan p = plan(a);
  AttnDev d = attn_dev<T>(a);
  use_workspace(d, a.workspace, p.slots, 16);
  d.max_parts = 1;
  d.blocks = a.blocks;
  d.block_count = static_cast<int>(a.block_count);
  d.width = static_cast<int>(a.c.table_width);
  d.parts = p.parts;
  d.by_parts = make_fastdiv(d.parts);
  const bool page16 = pages_of_16(a.c);
  // Work-items of a launch stay below 2^32.
  const int64_t items = p.row_tiles * p.parts, per_launch = std::max<int64_t>(1, (int64_t(1) << 22) / a.c.kv_heads);
  for (int64_t i0 = 0; i0 < items; i0 += per_launch) {
    d.item0 = static_cast<int>(i0);
    const dim3 grid(static_cast<unsigned>(std::min(per_launch, items - i0) * a.c.kv_heads)), block(kWaves * kWave);
    if (p.once) {
      if (page16) AKO_LAUNCH((attn_rows<T, MX, DP, kWaves, true, true, true>), grid, block, 0, stream, d);
      else AKO_LAUNCH((attn_rows<T, MX, DP, kWaves, false, true, true>), grid, block, 0, stream, d);
    } else {
      if (page16) AKO_LAUNCH((attn_rows<T, MX, DP, kWaves, true, false, true>), grid, block, 0, stream, d);
      else AKO_LAUNCH((attn_rows<T, MX, DP, kWaves, false, false, true>), grid, block, 0, stream, d);
    }
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  return p.parts == 1 ? hipSuccess : launch_attn_join(d, a.dtype, a.c.tokens * a.q_heads, 16, stream);
}

template <typename T, bool MX>
hipError_t by_head_dim(const PagedAttentionArgs& a, hipStream_t stream) {
  if (a.c.head_dim <= 64) return run<T, MX, 64>(a, stream);
  if (a.c.head_dim <= 128) return run<T, MX, 128>(a, stream);
  return run<T, MX, 256>(a, stream);
}

}  // namespace

int64_t paged_blocks_workspace(const PagedAttentionArgs& a) {
  const Plan p = plan(a);
  return p.parts == 1 ? 0 : workspace_bytes(a, p.slots, 16);
}

hipError_t launch_paged_blocks(const PagedAttentionArgs& a, hipStream_t stream) {
  switch (a.dtype) {
    case kF32: return a.c.mx ? by_head_dim<float, true>(a, stream) : by_head_dim<float, false>(a, stream);
    case kF16: return a.c.mx ? by_head_dim<_Float16, true>(a, stream) : by_head_dim<_Float16, false>(a, stream);
    case kBF16: return a.c.mx ? by_head_dim<__bf16, true>(a, stream) : by_head_dim<__bf16, false>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace ako

// What the attention kernels over a paged key/value cache share, and the kernel for up to
// 16 rows per workgroup (paged_attention.hip has the mathematics): the work items, the matrix
// products, the masks of what a row sees, and the joining of parts.
#pragma once

#include <algorithm>
#include <cmath>
#include <limits>

#include "paged.h"

namespace ako {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// The maximum of a row that sees keys but only scores of -infinity: 0 / 0, as its
// softmax says, where a row that sees nothing (its maximum -infinity) is zero.
constexpr float kAllInf = -std::numeric_limits<float>::max();
__device__ __forceinline__ float inverse_total(float m, float l) {
  return l != 0.0f ? 1.0f / l : m == -__builtin_inff() ? 0.0f : __builtin_nanf("");
}
// Whether a part of a row's keys has sums: those under scores of -infinity alone
// are 0, but 0 * NaN where a value is not finite.
__device__ __forceinline__ bool holds_sums(float m, float l) { return l != 0.0f || m != -__builtin_inff(); }

constexpr int kWaves = 4;          // of a workgroup
constexpr int kMaxParts = kWave;   // of a key range

struct AttnDev {
  PagedDev c;
  const void* q;
  void* out;
  // Parts of split key ranges: `slots` row tiles of unscaled sums, of maxima and
  // totals, and per output row the first part's row among those and the number of parts.
  float* part_o;
  float2* part_ml;
  int2* row_parts;
  int slots;
  int64_t qs[3];
  int q_heads, kv_heads, group, head_dim;
  int window, sinks;
  int item0;        // first work item of the launch
  int max_parts;    // 1: key ranges are not split
  int min_tiles;    // ranges of up to so many key tiles are not cut, and parts are at least so long,
  int few_tiles;    // or so long, where a launch has few items
  float per_item;   // 1 / work items wanted for each key head
  float per_few;    // 1 / items of a launch that is not worth cutting further, for each key head
  float scale_log2;       // |scale| * log2(e), above 0: exponentials are of base 2
  unsigned q_sign;        // sign bits to flip in a word of q (scale < 0)
  FastDiv by_kv_heads, by_group;
  // attn_rows over listed blocks: [tokens, kv_heads, block_count] numbers of pages of the sequence.
  const int* blocks;
  int block_count, width;
  int parts;        // of every row tile's keys
  FastDiv by_parts;
};

// The rows' outputs from the parts of their keys that the kernels have left (paged_attention.hip).
hipError_t launch_attn_join(const AttnDev& d, int dtype, int64_t rows, int tile, hipStream_t stream);

// What a call says of itself, but for how it is cut up.
template <typename T>
AttnDev attn_dev(const PagedAttentionArgs& a) {
  AttnDev d{};
  d.c = paged_dev(a.c);
  d.q = a.q;
  d.out = a.out;
  for (int i = 0; i < 3; ++i) d.qs[i] = a.qs[i];
  d.q_heads = static_cast<int>(a.q_heads);
  d.kv_heads = static_cast<int>(a.c.kv_heads);
  d.group = static_cast<int>(a.q_heads / a.c.kv_heads);
  d.head_dim = static_cast<int>(a.c.head_dim);
  // Not 0: times it a masked score, -inf, has to stay that.
  d.scale_log2 = std::max(std::fabs(a.scale) * 1.44269504088896340736f, std::numeric_limits<float>::min());
  d.q_sign = a.scale < 0.0f ? (sizeof(T) == 4 ? 0x80000000u : 0x80008000u) : 0u;
  d.by_kv_heads = make_fastdiv(d.kv_heads);
  d.by_group = make_fastdiv(d.group);
  return d;
}
// The parts' memory in a call's workspace: sums, maxima and totals of `slots` tiles of `rows` rows, then row_parts.
inline void use_workspace(AttnDev& d, void* space, int64_t slots, int rows) {
  d.part_o = static_cast<float*>(space);
  d.part_ml = reinterpret_cast<float2*>(d.part_o + slots * rows * d.head_dim);
  d.row_parts = reinterpret_cast<int2*>(d.part_ml + slots * rows);
  d.slots = static_cast<int>(slots);
}
inline int64_t workspace_bytes(const PagedAttentionArgs& a, int64_t slots, int rows) {
  return slots * rows * (a.c.head_dim + 2) * static_cast<int64_t>(sizeof(float)) +
         a.c.tokens * a.q_heads * static_cast<int64_t>(sizeof(int2));
}
// Whether PAGE16 (row_offsets) holds: rows' offsets inside 16 slots are 32-bit there.
inline bool pages_of_16(const PagedArgs& c) {
  bool page16 = c.page_size % 16 == 0;
  for (const auto* st : {c.kst, c.vst, c.ksst, c.vsst}) page16 = page16 && st[2] < (int64_t(1) << 24);
  return page16;
}

// The key tiles that a row tile sees, in order: those of the sinks, then those
// from the first row's window on.
struct KeyTiles {
  int sink_tiles, low, end;  // low: a multiple of the tile
  int count;
};
template <int KT>
__device__ __forceinline__ KeyTiles key_tiles(const AttnDev& a, int first_pos, int last_pos) {
  KeyTiles k{0, 0, 0, 0};
  k.end = min(last_pos + 1, a.c.capacity);
  if (k.end <= 0) return k;
  if (a.window > 0) {
    k.low = max(0, max(first_pos, 0) - a.window + 1) / KT * KT;
    k.low = min(k.low, k.end / KT * KT);
    k.sink_tiles = (min(a.sinks, k.low) + KT - 1) / KT;
  }
  k.count = k.sink_tiles + (k.end - k.low + KT - 1) / KT;
  return k;
}

// A work item: a tile of rows of one sequence (or of padding) that share a key
// head, and a part of the keys that they see.
struct Item {
  int seq;     // -1: padding, nothing is visible
  int token0;  // first token row of the sequence
  int rows;    // rows of the sequence for one key head
  int row0;    // the tile's first
  int pos0;    // position of token0, negative where the sequence is shorter than its rows
  int part, parts;
  int slot;    // of the parts' memory, for part 0 of key head 0
};

// Work item `item` of one key head. Items are laid out on the device, from the
// lengths that are only known there: with T the key tiles of all row tiles,
// a range of n > min_tiles tiles is cut into n / L parts, L = max(min_tiles, T * per_item),
// or as little as few_tiles as long as that makes few items (T * per_few): then the
// time is that of one item, and not of the bytes. That makes at most 1 / per_item
// items more than there are row tiles, which the host launches; long sequences do not hold up a step of short ones, and where all
// are long the items are 1 / per_item, a number of whole rounds of the chip
// (one item more would cost another round). What lies behind the last packed
// sequence counts as one more, padding. Sequences are looked at 64 at a time, one per lane,
// by every workgroup: at 64 keys and 8 key heads 64 sequences take 7.1 us, 256 29, 1024 165.
template <int R, int KT>
__device__ __forceinline__ bool find_item(const AttnDev& a, int item, Item& t) {
  const PagedDev& p = a.c;
  const int lane = threadIdx.x % kWave;
  const int n = p.cu ? p.n_seqs + 1 : p.seq > 0 ? p.n_seqs : 0;
  struct Seq { int token0, rows, pos0, row_tiles, tiles; };
  const auto look = [&](int i) {
    Seq s{0, 0, -1, 0, 0};
    if (i >= n) return s;
    if (p.cu == nullptr) {
      s.token0 = i * p.seq;
      s.rows = p.seq * a.group;
      s.pos0 = max(p.lens[i], 0) - p.seq;
    } else {
      s.token0 = min(max(p.cu[i], 0), p.tokens);
      const int end = i < p.n_seqs ? min(max(p.cu[i + 1], 0), p.tokens) : p.tokens;
      s.rows = max(0, end - s.token0) * a.group;
      s.pos0 = (i < p.n_seqs ? max(p.lens[i], 0) : -1) - max(0, end - s.token0);
    }
    s.row_tiles = (s.rows + R - 1) / R;
    if (s.row_tiles > 0)
      s.tiles = key_tiles<KT>(a, s.pos0 + static_cast<int>(fast_div((s.row_tiles - 1) * R, a.by_group)),
                              s.pos0 + static_cast<int>(fast_div(s.rows - 1, a.by_group))).count;
    return s;
  };
  Seq s = look(lane);
  int len = 1 << 30;
  if (a.max_parts > 1) {
    float total = static_cast<float>(s.row_tiles) * static_cast<float>(s.tiles);
    for (int base = kWave; base < n; base += kWave) {
      const Seq more = look(base + lane);
      total += static_cast<float>(more.row_tiles) * static_cast<float>(more.tiles);
    }
    // Rounded up past the float sum's own error, so that the items stay in bound.
    // 1e9 tiles are more than any range has.
    total = wave_sum(total) * 1.0001f;
    const auto share = [&](float per) { return static_cast<int>(__builtin_fminf(total * per, 1e9f)) + 1; };
    len = max(share(a.per_item), min(a.min_tiles, max(a.few_tiles, share(a.per_few))));
  }
  int before = 0, slots_before = 0;
  for (int base = 0; base < n; base += kWave) {
    if (base > 0) s = look(base + lane);
    const int parts = s.tiles > a.min_tiles ? min(a.max_parts, max(1, s.tiles / len)) : 1;
    const int items = s.row_tiles * parts, slots = parts > 1 ? items : 0;
    int upto = items, slots_upto = slots;
#pragma unroll
    for (int k = 1; k < kWave; k *= 2) {
      const int x = __shfl_up(upto, k), y = __shfl_up(slots_upto, k);
      if (lane >= k) {
        upto += x;
        slots_upto += y;
      }
    }
    const uint64_t behind = __ballot(item < before + upto);
    if (behind) {
      const int l = __builtin_ctzll(behind);
      t.parts = __builtin_amdgcn_readlane(parts, l);
      t.token0 = __builtin_amdgcn_readlane(s.token0, l);
      t.rows = __builtin_amdgcn_readlane(s.rows, l);
      t.pos0 = __builtin_amdgcn_readlane(s.pos0, l);
      t.seq = p.cu && base + l >= p.n_seqs ? -1 : base + l;
      const int local = item - before - __builtin_amdgcn_readlane(upto - items, l);
      // The last rows first: they see the most keys.
      const int from_last = local / t.parts;
      t.row0 = (__builtin_amdgcn_readlane(s.row_tiles, l) - 1 - from_last) * R;
      t.part = local - from_last * t.parts;
      t.slot = slots_before + __builtin_amdgcn_readlane(slots_upto - slots, l) + from_last * t.parts;
      // Indexes that make no sense may have wrapped the sums.
      return local >= 0 && t.row0 >= 0 &&
             (t.parts == 1 || (t.slot >= 0 && (int64_t(t.slot) + t.parts) * a.kv_heads <= a.slots));
    }
    before += __builtin_amdgcn_readlane(upto, kWave - 1);
    slots_before += __builtin_amdgcn_readlane(slots_upto, kWave - 1);
  }
  return false;
}

// ---- matrix products ----------------------------------------------------------
// Sixteen rows of A times sixteen columns of B, a packet of 16 bytes of the inner
// dimension per lane. kShift: weights (and so totals and sums) are held times
// 2^kShift; a power of two that the final division removes. fp16's weights
// would be subnormal, with fewer bits, below 2^-14 of the largest; times 2^15
// the largest is still far from fp16's end and the last bit is lost below 2^-29.
template <typename T> struct Mfma;
template <> struct Mfma<__bf16> {
  static constexpr float kShift = 0.0f;
  static __device__ __forceinline__ f32x4 mul(const Pack<__bf16, 8>& a, const Pack<__bf16, 8>& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a.raw), __builtin_bit_cast(bf16x8, b.raw), c, 0, 0, 0);
  }
};
template <> struct Mfma<_Float16> {
  static constexpr float kShift = 15.0f;
  static __device__ __forceinline__ f32x4 mul(const Pack<_Float16, 8>& a, const Pack<_Float16, 8>& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a.raw), __builtin_bit_cast(f16x8, b.raw), c, 0, 0, 0);
  }
};
template <> struct Mfma<float> {
  static constexpr float kShift = 0.0f;
  static __device__ __forceinline__ f32x4 mul(const Pack<float, 4>& a, const Pack<float, 4>& b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.e[i], b.e[i], c, 0, 0, 0);
    return c;
  }
};

__device__ __forceinline__ float max_over_groups(float v) {  // over the lanes l % 16
  v = __builtin_fmaxf(v, __shfl_xor(v, 16));
  return __builtin_fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float max_of_halves(float v) {  // over the lanes l % 32
  const unsigned x = __builtin_bit_cast(unsigned, v);
  const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return __builtin_fmaxf(__builtin_bit_cast(float, static_cast<unsigned>(r[0])), __builtin_bit_cast(float, static_cast<unsigned>(r[1])));
}
__device__ __forceinline__ float sum_over_groups(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// Nonzero where a word of values holds an infinity or NaN (or might, once
// multiplied by its scale): their exponents are all ones, and one more in the exponent's
// last place then carries into the sign's, which was masked out. e4m3 has only NaN,
// all ones below the sign; scales from 2^8 on in fp16, from 2^120 on in the other types,
// can take it past the end, and under code 255 everything is NaN, zeros too.
template <typename T, bool MX>
__device__ __forceinline__ unsigned odd_values(u32x4 w, unsigned code) {
  constexpr unsigned kMask = MX ? 0x7f7f7f7fu : sizeof(T) == 4 ? 0x7f800000u : __is_same(T, __bf16) ? 0x7f807f80u : 0x7c007c00u;
  constexpr unsigned kOne = MX ? 0x01010101u : sizeof(T) == 4 ? 0x00800000u : __is_same(T, __bf16) ? 0x00800080u : 0x04000400u;
  constexpr unsigned kSign = MX ? 0x80808080u : sizeof(T) == 4 ? 0x80000000u : 0x80008000u;
  unsigned odd = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) odd |= (w[i] & kMask) + kOne;
  odd &= kSign;
  if constexpr (MX) odd |= code >= (__is_same(T, _Float16) ? 127 + 8 : 127 + 120);
  return odd;
}

// Orders LDS accesses of one wavefront's lanes to each other's data. The LDS
// serves a wavefront in order; only the compiler has to be held.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Infinities and NaN among values that not every row sees: a weight of 0 would
// not cancel them. They are taken out of V (zeros in their places), and for
// each of the head's elements two words of `masks` (DP of them, then DP more) tell which of a
// wavefront's keys held +infinity and which -infinity there, NaN in both. A row
// then adds the infinities of those keys that it does see (add_odd).
// Bit n * KPW + w is the key of load n that is w-th among the KPW of the wavefront.
template <typename T, bool MX, int DP, int KPW, int LOADS>
__device__ __forceinline__ void take_out_odd(u32x4 (&v)[LOADS], unsigned (&code)[LOADS], unsigned* masks, int lane) {
  constexpr int C = MX ? 16 : 16 / static_cast<int>(sizeof(T)), LANES = DP / C;
  const int part = lane % LANES;
  for (int i = lane; i < 2 * DP; i += kWave) masks[i] = 0;
  wave_fence();
#pragma unroll
  for (int n = 0; n < LOADS; ++n) {
#pragma unroll
    for (int e = 0; e < C; ++e) {
      __builtin_amdgcn_sched_barrier(0);  // rare: element by element, to cost the loop around it no registers
      constexpr int kBits = 128 / C, kPerWord = 32 / kBits;  // of an element of v[n]
      const unsigned word = v[n][e / kPerWord], shift = e % kPerWord * kBits;
      float f;
      if constexpr (MX) f = to_f32(FromE4m3<T>::lo(word >> shift, e8m0_scale(code[n]))[0]);
      else if constexpr (sizeof(T) == 4) f = __builtin_bit_cast(float, word);
      else f = to_f32(__builtin_bit_cast(T, static_cast<unsigned short>(word >> shift)));
      if (__builtin_fabsf(f) < __builtin_inff()) continue;
      const unsigned bit = 1u << (n * KPW + lane / LANES);
      if (!(f < 0.0f)) atomicOr(&masks[part * C + e], bit);
      if (!(f > 0.0f)) atomicOr(&masks[DP + part * C + e], bit);
      const unsigned all = kBits == 32 ? ~0u : ((1u << (kBits % 32)) - 1) << shift;
      v[n][e / kPerWord] = word & ~all;
    }
    if (MX && code[n] == 255) code[n] = kUnitCode;
  }
}

// Adds to elements e .. e + 3 the infinities that a row sees.
__device__ __forceinline__ float odd_sum(unsigned plus, unsigned minus) {
  return (plus ? __builtin_inff() : 0.0f) - (minus ? __builtin_inff() : 0.0f);
}
template <int DP>
__device__ __forceinline__ f32x4 odd_sums(const unsigned* masks, int e, unsigned seen) {
  const u32x4 p = *reinterpret_cast<const u32x4*>(masks + e), m = *reinterpret_cast<const u32x4*>(masks + DP + e);
  f32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = odd_sum(p[i] & seen, m[i] & seen);
  return r;
}

// The keys of a tile of up to 64, from k0 on, that a row sees of those that are
// there: j <= hi, and j >= lo or j < sinks.
__device__ __forceinline__ uint64_t below(int n) {
  return n <= 0 ? 0 : n >= 64 ? ~uint64_t(0) : (uint64_t(1) << n) - 1;
}
__device__ __forceinline__ uint64_t keys_seen(uint64_t there, int k0, int lo, int hi, int sinks) {
  return there & below(hi + 1 - k0) & (~below(lo - k0) | below(sinks - k0));
}

// Where a tile's rows lie: lane j finds the byte offsets of key j's rows once for
// the tile, and a load takes them from there. `mine` is a lane's key among the
// KPW consecutive ones that a load covers, from the tile's key `at` on.
//
// PAGE16 (pages of a multiple of 16 slots; KPW divides 16): a load's keys lie in
// one page, so its address is scalar, that of key `at`, and lanes add a 32-bit
// offset that is the same for every tile. Slots past `end` inside a page are
// read with it; blocks of 16 keys past `end` are read as the last block. Otherwise
// each lane takes its own key's offset, and keys past `end` are read as the
// last. Absent pages are read as page 0. Every address is inside the pool.
template <bool MX>
struct RowOffsets {
  int64_t k, v, ks, vs;
};
template <typename T, bool MX, bool PAGE16>
__device__ __forceinline__ RowOffsets<MX> row_offsets(const PagedDev& c, int page, int key, int end) {
  constexpr int EB = MX ? 1 : sizeof(T);
  if constexpr (PAGE16) key = key < end ? key : (end - 1) / 16 * 16 + key % 16;
  else key = min(key, end - 1);
  const int slot = key - static_cast<int>(fast_div(key, c.by_page)) * c.page_size;
  page = page >= 0 && page < c.num_pages ? page : 0;
  RowOffsets<MX> r;
  r.k = (page * c.kst[0] + slot * c.kst[2]) * EB;
  r.v = (page * c.vst[0] + slot * c.vst[2]) * EB;
  if constexpr (MX) {
    r.ks = page * c.ksst[0] + slot * c.ksst[2];
    r.vs = page * c.vsst[0] + slot * c.vsst[2];
  }
  return r;
}
template <bool PAGE16>
__device__ __forceinline__ int64_t offset_at(int64_t offsets, int at, int mine) {
  const int lo = static_cast<int>(offsets), hi = static_cast<int>(offsets >> 32);
  unsigned l;
  int h;
  if constexpr (PAGE16) {
    l = __builtin_amdgcn_readlane(lo, at);
    h = __builtin_amdgcn_readlane(hi, at);
  } else {
    l = __shfl(lo, at + mine);
    h = __shfl(hi, at + mine);
  }
  return static_cast<int64_t>(static_cast<uint64_t>(static_cast<unsigned>(h)) << 32 | l);
}

// A key head's part of the pools.
struct HeadPools {
  const uint8_t *k, *v, *ks, *vs;
};
template <typename T, bool MX>
__device__ __forceinline__ HeadPools head_pools(const PagedDev& c, int head) {
  constexpr int EB = MX ? 1 : sizeof(T);
  return HeadPools{static_cast<const uint8_t*>(c.k) + head * c.kst[1] * EB, static_cast<const uint8_t*>(c.v) + head * c.vst[1] * EB,
                   MX ? c.ks + head * c.ksst[1] : nullptr, MX ? c.vs + head * c.vsst[1] : nullptr};
}

// Sixteen bytes of a row of T (or, MX, of e4m3), aligned as its elements are.
// ONCE: rows that no other workgroup reads, with the non-temporal hint.
template <typename T, bool MX, bool ONCE>
__device__ __forceinline__ u32x4 load16(const uint8_t* p) {
  if constexpr (MX) return load_pack<uint8_t, 16, ONCE>(p).raw;
  else return load_pack<T, 16 / static_cast<int>(sizeof(T)), ONCE>(reinterpret_cast<const T*>(p)).raw;
}

// ---- up to 16 rows per workgroup -------------------------------------------------
// Decode steps, where the cache's bytes are all that counts, and every step in
// 32 bits. A wavefront takes key tiles of its own, loads whole rows of K and V
// (a kilobyte per instruction) into registers and from there into its own
// piece of LDS, so that no barrier stands in the loop; the loads of a later tile
// are issued as soon as those registers are free, and are in flight while this
// tile is worked on. The wavefronts' results are joined in LDS at the end.
//
// Bound by HBM once the ranges are long: 2.1 GB of e4m3 pages in 341 us, 6.2 TB/s, 538 MB
// of fp16 under a window in 90 us, 6.0 TB/s (a large copy reaches 6.67); what is
// fetched is within 1.5% of the keys and values seen. Whole rows of K through
// LDS rather than the operand's 16 bytes of 16 rows per load, and non-temporal
// loads, took the first from 5.6 TB/s. The 8-bit tiles are half as large, so
// two of them are in flight. Short ranges are latency: 11 us at 640 keys, of
// which 4 are the join's.
template <typename T, bool MX, int DP>
struct RowsShape {
  static constexpr int kBlocks = sizeof(T) == 4 ? 1 : 2;    // 16-key blocks per tile
  static constexpr int kKeys = 16 * kBlocks;
  static constexpr int kChunk = MX ? 16 : 16 / sizeof(T);   // elements in 16 loaded bytes
  static constexpr int kRowLanes = DP / kChunk;             // lanes across a row
  static constexpr int kRowKeys = kWave / kRowLanes;        // keys per load
  static constexpr int kLoads = kKeys / kRowKeys;           // of K and of V, per lane and tile
  static constexpr int kAhead = MX ? 2 : 1;                 // tiles in flight
  static constexpr int kRowBytes = DP * sizeof(T);
  static constexpr int kTileBytes = kKeys * kRowBytes;      // = 16 rows of DP floats, too
};

// LDS place of 16-byte packet p of key's row. Rows are multiples of 128 or 256
// bytes, all on the same banks: packets are exchanged in pairs (a transposing
// read takes 32 bytes of four keys' rows) so that eight keys' pairs lie on
// different banks.
template <int ROW_BYTES>
__device__ __forceinline__ int lds_packet(int key, int p) {
  constexpr int kPairs = ROW_BYTES / 32;
  const int x = kPairs >= 8 ? key & 7 : (key >> 1) & (kPairs - 1);
  return key * ROW_BYTES + ((p ^ (x << 1)) << 4);
}

// LDS place of packet p of a key's row of K, which is read 16 bytes of 32 rows at a
// time: sixteen rows' packets lie on different banks.
template <int ROW_BYTES>
__device__ __forceinline__ int lds_packet_k(int key, int p) {
  constexpr int kPackets = ROW_BYTES / 16;
  const int x = kPackets >= 16 ? key & 15 : (key >> 1) & (kPackets - 1);
  return key * ROW_BYTES + ((p ^ x) << 4);
}

//
// BLOCKS: each row sees only the blocks (pages) listed for its token and key head, and of
// those what its position lets it see. A tile's tokens are done together: the blocks
// that any of them lists are found as a set (a word of LDS for each block, in which each token
// sets its bit), a segment of blocks at a time, and key tiles run over the positions of the
// blocks found, laid end to end. So a block that several of them list is read once, blocks may be listed in any order
// and more than once, and small pages leave no gaps in a tile.
constexpr int kSegment = 1024;  // blocks

template <typename T, bool MX, int DP, int WAVES, bool PAGE16, bool ONCE, bool BLOCKS>
__global__ __launch_bounds__(WAVES* kWave, DP * sizeof(T) <= 128 && !MX ? 3 : DP * sizeof(T) <= 256 ? 2 : 1) void attn_rows(AttnDev a) {
  using S = RowsShape<T, MX, DP>;
  constexpr int KT = S::kKeys, NB = S::kBlocks, C = S::kChunk, NV = S::kLoads, AHEAD = S::kAhead;
  constexpr int E = 16 / static_cast<int>(sizeof(T));  // elements of an LDS packet
  __shared__ __align__(16) unsigned char lds[WAVES][2][S::kTileBytes];  // K and V
  __shared__ float2 lds_ml[WAVES][16];
  __shared__ __align__(16) unsigned lds_odd[WAVES][2 * DP];
  // BLOCKS: of each block of the segment the tokens that list it; then those blocks, a block's number
  // in the segment below its tokens' bits.
  [[maybe_unused]] __shared__ unsigned lds_tokens[BLOCKS ? kSegment : 1], lds_blocks[BLOCKS ? kSegment : 1];
  [[maybe_unused]] __shared__ int lds_next;  // the first listed block behind the segment
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const int col = lane % 16, g = lane / 16;
  unsigned char* const kl = lds[wave][0];
  unsigned char* const vt = lds[wave][1];

  // Key heads run fastest over the workgroups, so that the XCDs share them out
  // and the row tiles of one head meet in one XCD's L2.
  const unsigned nth = fast_div(blockIdx.x, a.by_kv_heads);
  const int kvh = blockIdx.x - nth * a.kv_heads;
  Item t;
  if constexpr (BLOCKS) {
    const unsigned item = a.item0 + nth, tile = fast_div(item, a.by_parts);
    if (!find_item<16, KT>(a, tile, t)) return;
    t.parts = a.parts;
    t.part = item - tile * a.parts;
    t.slot = tile * a.parts;
  } else {
    if (!find_item<16, KT>(a, a.item0 + nth, t)) return;
  }

  const int live = min(16, t.rows - t.row0);
  const int my_token = fast_div(t.row0 + col, a.by_group);  // of the sequence
  const int my_head = kvh * a.group + (t.row0 + col - my_token * a.group);
  const int first_pos = t.pos0 + static_cast<int>(fast_div(t.row0, a.by_group));
  const int last_pos = t.pos0 + static_cast<int>(fast_div(t.row0 + live - 1, a.by_group));
  const KeyTiles kt = t.seq < 0 ? KeyTiles{0, 0, 0, 0} : key_tiles<KT>(a, first_pos, last_pos);
  const int begin = static_cast<int>(static_cast<int64_t>(kt.count) * t.part / t.parts);
  int end = static_cast<int>(static_cast<int64_t>(kt.count) * (t.part + 1) / t.parts);

  // BLOCKS: the tile's tokens, of the sequence, and the segment that is worked on: its first block, and the positions
  // of its listed blocks.
  [[maybe_unused]] const int token_first = fast_div(t.row0, a.by_group);
  [[maybe_unused]] const int tokens = static_cast<int>(fast_div(t.row0 + live - 1, a.by_group)) - token_first + 1;
  [[maybe_unused]] int segment = 0, listed = 0;
  // BLOCKS: whether to look for infinities and NaN among the values. Nearly every tile has keys that some row does not
  // see, and the look is a quarter of a tile's vector instructions; without it they turn up in the sums, as NaN where
  // the weight is 0, and all is done again with the look (2048 tokens of 1024 of 32768 keys: 452 us with the look, 420 without).
  [[maybe_unused]] bool look = false;

  // This lane's query row, in the order of the K operand.
  const bool row_live = col < live;
  const int hi = row_live ? t.pos0 + my_token : -1;
  const int lo = a.window > 0 ? max(0, max(hi, 0) - a.window + 1) : 0;
  constexpr int NQ = DP / (4 * E);  // packets of the row in this lane: elements (4 c + g) E ..
  Pack<T, E> q[NQ];
  {
    const int b = a.c.cu ? 0 : t.seq;
    const T* x = static_cast<const T*>(a.q) + b * a.qs[0] + (t.token0 - b * a.c.seq + my_token) * a.qs[1] + my_head * a.qs[2];
#pragma unroll
    for (int c = 0; c < NQ; ++c) {
      const int d = (4 * c + g) * E;
      q[c].raw = u32x4{0, 0, 0, 0};
      if (row_live && d < a.head_dim) q[c] = load_pack<T, E>(x + d);
      q[c].raw ^= a.q_sign;
    }
  }

  float m = -__builtin_inff(), l = 0.0f;
  f32x4 o[DP / 16];
#pragma unroll
  for (int i = 0; i < DP / 16; ++i) o[i] = f32x4{0, 0, 0, 0};

  const int* const table = a.c.table + (t.seq < 0 ? 0 : t.seq * a.c.table_stride);
  const auto tile_start = [&](int i) {
    return i < kt.sink_tiles ? i * KT : kt.low + (i - kt.sink_tiles) * KT;
  };
  // BLOCKS: the key of lane j in tile i as its place among the segment's listed positions (keys past the
  // end as row_offsets takes them), and its block's entry in the list.
  [[maybe_unused]] const auto listed_place = [&](int i) {
    const int v = i * KT + lane % KT;
    return v < listed ? v : PAGE16 ? (listed - 1) / 16 * 16 + v % 16 : listed - 1;
  };
  [[maybe_unused]] const auto listed_block = [&](int place) { return lds_blocks[fast_div(place, a.c.by_page)]; };
  [[maybe_unused]] const auto listed_key = [&](int place) {  // its position
    const int nth = fast_div(place, a.c.by_page);
    return (segment + static_cast<int>(lds_blocks[nth] & 0xffffu) - nth) * a.c.page_size + place;
  };
  // Lane j holds the page of the tile's key j (keys past the end: of the last one).
  const auto look_up = [&](int i) {
    if constexpr (BLOCKS) return table[segment + static_cast<int>(listed_block(listed_place(i)) & 0xffffu)];
    else return table[fast_div(min(tile_start(i) + lane % KT, kt.end - 1), a.c.by_page)];
  };

  // Loaded bytes of a tile, and which of its keys are there.
  struct Loaded {
    u32x4 k[NV], v[NV];
    unsigned kcode[NV], vcode[NV];
    unsigned there;
  };
  constexpr int EB = MX ? 1 : sizeof(T);
  const int vkey = lane / S::kRowLanes, vpart = lane % S::kRowLanes;
  const bool part_in = vpart * C < a.head_dim;
  const int pd = part_in ? vpart * C : 0;
  const unsigned koff = ((PAGE16 ? vkey * static_cast<unsigned>(a.c.kst[2]) : 0) + pd) * EB;
  const unsigned voff = ((PAGE16 ? vkey * static_cast<unsigned>(a.c.vst[2]) : 0) + pd) * EB;
  const unsigned kcoff = (PAGE16 ? vkey * static_cast<unsigned>(a.c.ksst[2]) : 0) + pd / 32;
  const unsigned vcoff = (PAGE16 ? vkey * static_cast<unsigned>(a.c.vsst[2]) : 0) + pd / 32;
  const HeadPools pools = head_pools<T, MX>(a.c, kvh);
  const auto load = [&](Loaded& x, int i, int pages) __attribute__((always_inline)) {
    const int k0 = BLOCKS ? i * KT : tile_start(i);
    // Pages laid end to end: a place's slot is a position's.
    const RowOffsets<MX> r = row_offsets<T, MX, PAGE16>(a.c, pages, k0 + lane % KT, BLOCKS ? listed : kt.end);
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int at = n * S::kRowKeys;
      x.k[n] = load16<T, MX, ONCE>(pools.k + offset_at<PAGE16>(r.k, at, vkey) + koff);
      x.v[n] = load16<T, MX, ONCE>(pools.v + offset_at<PAGE16>(r.v, at, vkey) + voff);
      if constexpr (MX) {
        x.kcode[n] = (pools.ks + offset_at<PAGE16>(r.ks, at, vkey))[kcoff];
        x.vcode[n] = (pools.vs + offset_at<PAGE16>(r.vs, at, vkey))[vcoff];
      }
    }
    bool there = pages >= 0 && pages < a.c.num_pages && lane < KT && k0 + lane < (BLOCKS ? listed : kt.end);
    if constexpr (BLOCKS) there = there && listed_key(listed_place(i)) <= last_pos;
    x.there = static_cast<unsigned>(__ballot(there));
  };
  // Packet `part` of a row into LDS, as T.
  const auto to_lds = [&](u32x4 w, unsigned code, auto place) {
    if constexpr (MX) {
      const float s = e8m0_scale(code);
      const Eight<T> x = from_e4m3<T>(u32x2{w[0], w[1]}, s), y = from_e4m3<T>(u32x2{w[2], w[3]}, s);
#pragma unroll
      for (int h = 0; h < 16 / E; ++h)
        *reinterpret_cast<u32x4*>(place(vpart * (16 / E) + h)) = h * E < 8 ? x.p[h * E % 8 / E].raw : y.p[h * E % 8 / E].raw;
    } else {
      *reinterpret_cast<u32x4*>(place(vpart)) = w;
    }
  };

  Loaded loaded[AHEAD];
  unsigned any = 0;  // nonzero where the row sees a key
  int pages = 0;  // of the next tile to load
  const auto take_out_missing = [&](Loaded& x) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      if (!(x.there >> (n * S::kRowKeys + vkey) & 1)) {
        x.v[n] = u32x4{0, 0, 0, 0};
        x.vcode[n] = kUnitCode;
      }
    }
  };
  const auto work = [&](Loaded& x, int i) __attribute__((always_inline)) {
    const unsigned here = x.there;
    // Whether every live row sees every key of the tile, and the keys that this lane's row sees.
    constexpr unsigned kAll = KT == 32 ? ~0u : 0xffffu;
    bool whole;
    unsigned seen;
    if constexpr (BLOCKS) {
      const int place = listed_place(i), key = listed_key(place);
      const unsigned by = listed_block(place) >> 16;
      whole = here == kAll && (static_cast<unsigned>(__ballot(by + 1 == 1u << tokens && key <= first_pos)) & kAll) == kAll;
      seen = whole ? ~0u : 0;
      if (!whole) {
        for (int n = 0; n < tokens; ++n) {
          const unsigned some = static_cast<unsigned>(__ballot((by >> n & 1) && key <= first_pos + n)) & here;
          if (row_live && my_token == token_first + n) seen = some;
        }
      }
    } else {
      const int k0 = tile_start(i);
      whole = here == kAll && k0 + KT - 1 <= first_pos && (a.window <= 0 || k0 > last_pos - a.window || k0 + KT <= a.sinks);
      seen = whole ? ~0u : static_cast<unsigned>(keys_seen(here, k0, lo, hi, a.sinks));
    }
    any |= seen;

    // K and V into LDS; rows of V that are not there as zeros.
    wave_fence();
    unsigned odd = 0;  // values that a weight of 0 would not cancel
    if (BLOCKS && !look && here != kAll) take_out_missing(x);
    if (BLOCKS ? look && !whole : !whole) {
      take_out_missing(x);
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        odd |= odd_values<T, MX>(x.v[n], MX ? x.vcode[n] : 0);
      }
      odd = __ballot(odd != 0) != 0;
      if (__builtin_expect(odd, 0)) take_out_odd<T, MX, DP, S::kRowKeys, NV>(x.v, x.vcode, lds_odd[wave], lane);
    }
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int key = n * S::kRowKeys + vkey;
      if (a.head_dim != DP && !part_in) x.k[n] = u32x4{0, 0, 0, 0};
      to_lds(x.k[n], MX ? x.kcode[n] : 0, [&](int p) { return kl + lds_packet_k<S::kRowBytes>(key, p); });
      to_lds(x.v[n], MX ? x.vcode[n] : 0, [&](int p) { return vt + lds_packet<S::kRowBytes>(key, p); });
    }
    const int step = BLOCKS ? t.parts * WAVES : WAVES;
    if (i + AHEAD * step < end) {
      // Loads return in order: the pages of the tile behind it are asked for
      // first, so that using them does not wait for the tile.
      const int now = pages;
      if (i + (AHEAD + 1) * step < end) pages = look_up(i + (AHEAD + 1) * step);
      load(x, i + AHEAD * step, now);
    }
    wave_fence();
    // S^T: block b holds keys k0 + 16 b + 4 g + r of query `col`.
    f32x4 s[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      s[b] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < NQ; ++c) {
        Pack<T, E> k;
        k.raw = *reinterpret_cast<const u32x4*>(kl + lds_packet_k<S::kRowBytes>(16 * b + col, 4 * c + g));
        s[b] = Mfma<T>::mul(k, q[c], s[b]);
      }
    }

    float top = -__builtin_inff();
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float v = s[b][r] * a.scale_log2;
        if (!whole) v = seen >> (16 * b + 4 * g + r) & 1 ? v : -__builtin_inff();
        s[b][r] = v;
        top = __builtin_fmaxf(top, v);
      }
    }
    const float mn = __builtin_fmaxf(m, max_over_groups(top));
    const float base = mn == -__builtin_inff() ? 0.0f : mn;
    if (__ballot(mn != m)) {
      const float keep = __builtin_amdgcn_exp2f(m - base);
      l *= keep;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) o[d] *= keep;
      m = mn;
    }
    // The second product takes the weights in the rows' type, as its matrix instruction does: each is rounded once, by up to
    // half a step of that type, as the output is after it. 2048 tokens of 1024 listed keys in bfloat16 are 1.72e-3 of
    // their size from 64 bits, with 32-bit weights 1.68e-3. The weights' own sum takes them in 32 bits.
    const float from = base - Mfma<T>::kShift;
    Pack<T, E> p;
    float pf[NB][4];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        pf[b][r] = __builtin_amdgcn_exp2f(s[b][r] - from);
        l += pf[b][r];
        if constexpr (E == 8) p.e[4 * b + r] = from_f32<T>(pf[b][r]);
        else p.e[r] = pf[b][r];
      }

    // O^T += V^T P^T.
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) {
      if constexpr (E == 8) {
        // Lane i of 16 gives the address of 8 bytes (key i / 4, elements 4 (i % 4) ..) and receives column i of the four keys.
        const int at = 16 * d + 4 * (col % 4), key = 4 * g + col / 4;
        u32x2 half[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b)
          half[b] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) s16x4*)(vt + lds_packet<S::kRowBytes>(16 * b + key, at / 8) + at % 8 * 2)));
        Pack<T, E> v;
        v.raw = u32x4{half[0][0], half[0][1], half[NB - 1][0], half[NB - 1][1]};
        o[d] = Mfma<T>::mul(v, p, o[d]);
      } else {
        Pack<T, E> v;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int e = 16 * d + col;
          v.e[r] = *reinterpret_cast<const T*>(vt + lds_packet<S::kRowBytes>(4 * g + r, e / E) + e % E * sizeof(T));
        }
        o[d] = Mfma<T>::mul(v, p, o[d]);
      }
    }
    if (__builtin_expect(odd, 0)) {
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) o[d] += odd_sums<DP>(lds_odd[wave], 16 * d + 4 * g, seen);
    }
  };

  // Key tiles first, first + STEP, ... below `end`.
  const auto walk = [&](int first, int step) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < AHEAD; ++n)
      if (first + n * step < end) {
        const int now = n == 0 ? look_up(first) : pages;
        if (first + (n + 1) * step < end) pages = look_up(first + (n + 1) * step);
        load(loaded[n], first + n * step, now);
      }
    for (int i = first; i < end; i += AHEAD * step) {
      work(loaded[0], i);
      if constexpr (AHEAD == 2)
        if (i + step < end) work(loaded[1], i + step);
    }
  };
  if constexpr (BLOCKS) {
    // The parts' wavefronts take the listed tiles in turn, over all segments.
    const int among = t.parts * WAVES, me = t.part * WAVES + wave;
    const int limit = t.seq < 0 || last_pos < 0 ? 0 : min(static_cast<int>(fast_div(last_pos, a.c.by_page)) + 1, a.c.capacity > 0 ? a.width : 0);
    int before = 0;  // tiles of earlier segments, modulo the wavefronts
    for (;;) {
      while (segment < limit) {
        for (int i = threadIdx.x; i < kSegment; i += WAVES * kWave) lds_tokens[i] = 0;
        if (threadIdx.x == 0) lds_next = limit;
        __syncthreads();
        int next = limit;
        for (int n = 0; n < tokens; ++n) {
          const int pos = first_pos + n;
          const int* const list = a.blocks + (int64_t(t.token0 + token_first + n) * a.kv_heads + kvh) * a.block_count;
          for (int i = threadIdx.x; i < a.block_count; i += WAVES * kWave) {
            const int b = list[i];
            // A block up to the token's own, by positions: b * page_size <= pos.
            if (b < segment || b >= limit || pos < 0 || b > static_cast<int>(fast_div(pos, a.c.by_page))) continue;
            if (b - segment < kSegment) atomicOr(&lds_tokens[b - segment], 1u << n);
            else next = min(next, b);
          }
        }
        if (next < limit) atomicMin(&lds_next, next);
        __syncthreads();
        int found = 0;
#pragma unroll 1
        for (int n = 0; n < kSegment / kWave; ++n) {
          const unsigned by = lds_tokens[n * kWave + lane];
          const uint64_t some = __ballot(by != 0);
          if (by != 0 && n % WAVES == wave)
            lds_blocks[found + __popcll(some & ((uint64_t(1) << lane) - 1))] = by << 16 | static_cast<unsigned>(n * kWave + lane);
          found += __popcll(some);
        }
        __syncthreads();
        listed = found * a.c.page_size;
        end = static_cast<int>(ceil_div(listed, KT));
        const int ahead = me - before;
        if (listed > 0) walk(ahead < 0 ? ahead + among : ahead, among);
        before = (before + end) % among;
        segment = lds_next;
        __syncthreads();
      }
      float worst = 0.0f;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) worst = __builtin_fabsf(o[d][r]) < __builtin_inff() ? worst : 1.0f;
      if (look || !__syncthreads_or(worst != 0.0f)) break;
      look = true;
      segment = before = 0;
      m = -__builtin_inff();
      l = 0.0f;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) o[d] = f32x4{0, 0, 0, 0};
    }
  } else {
    walk(begin + wave, WAVES);
  }

  wave_fence();
  // Join the wavefronts: o as rows of DP floats in the wavefront's own LDS, 16-byte
  // packets exchanged by the row's number against bank conflicts.
  l = sum_over_groups(l);
  if (any && m == -__builtin_inff()) m = kAllInf;
  if (g == 0) lds_ml[wave][col] = float2{m, l};
  float* const mine = reinterpret_cast<float*>(vt);
#pragma unroll
  for (int d = 0; d < DP / 16; ++d) *reinterpret_cast<f32x4*>(mine + col * DP + (((4 * d + g) ^ col) << 2)) = o[d];
  __syncthreads();
  for (int n = threadIdx.x; n < 16 * DP / 4; n += WAVES * kWave) {
    const int row = n / (DP / 4), d = n % (DP / 4) * 4;
    if (row >= live || d >= a.head_dim) continue;
    float M = -__builtin_inff(), L = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) M = __builtin_fmaxf(M, lds_ml[w][row].x);
    const float base = M == -__builtin_inff() ? 0.0f : M;
    f32x4 x = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float keep = __builtin_amdgcn_exp2f(lds_ml[w][row].x - base);
      L += lds_ml[w][row].y * keep;
      const f32x4 y = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds[w][1]) + row * DP + (((d / 4) ^ row) << 2));
      x += y * keep;  // zeros of a wavefront without keys; 0 * NaN where its scores were all -infinity
    }
    const int token = fast_div(t.row0 + row, a.by_group);
    const int64_t at = int64_t(t.token0 + token) * a.q_heads + kvh * a.group + (t.row0 + row - token * a.group);
    const int slot_row = ((t.slot + t.part) * a.kv_heads + kvh) * 16 + row;
    if ((BLOCKS ? t.parts : a.max_parts) > 1 && t.part == 0 && d == 0) a.row_parts[at] = int2{slot_row, t.parts};
    if (t.parts > 1) {
      if (d == 0) a.part_ml[slot_row] = float2{M, L};
      if (holds_sums(M, L)) *reinterpret_cast<f32x4*>(a.part_o + int64_t(slot_row) * a.head_dim + d) = x;
    } else {
      const float inv = inverse_total(M, L);
      Pack<T, 4> y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y.e[e] = from_f32<T>(x[e] * inv);
      store_pack<T, 4>(static_cast<T*>(a.out) + at * a.head_dim + d, y);
    }
  }
}

}  // namespace ako

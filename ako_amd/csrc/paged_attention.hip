// Attention of a step's tokens over a paged key/value cache on gfx950.
//
// Token row t at position p of its sequence sees the keys j <= p, and with a
// window w only those with j > p - w or j < sinks:
//   out = sum_j e^(scale q.k_j - m) v_j / sum_j e^(scale q.k_j - m),  m = max_j scale q.k_j
// in 32 bits, zero where nothing is visible. Keys are walked once, in tiles,
// with a running maximum m, total l and weighted sum o (rescaled by e^(m_old - m_new)
// where a tile raises m). The query rows of the heads that share a key head
// are laid side by side, row r = (token of the sequence) * group + (head in group),
// so that a tile of rows reads each key once for all of them.
//
// Products are formed transposed, S^T = K Q^T and O^T = V^T P^T: a lane then
// holds scores of one query only, its maximum and total are one lane's
// numbers, and the scores as they come out of the first product are the
// operand of the second without moving between lanes. The matrix
// instruction's k index is only a name for a key, so it is named by where the
// first product leaves its scores; V^T is read with the same names. V^T comes
// from rows of V in LDS through transposing reads.
//
// Weights e^(..) are at most 1 and are rounded to the rows' type for the second
// product (half a step each, as the result is); totals add the 32-bit
// weights. Long key ranges are split over workgroups and joined by a second
// kernel in order of the split, so results do not depend on scheduling.

#include <algorithm>
#include <cmath>
#include <limits>

#include "paged.h"

namespace ako {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

PagedTuning g_paged_tuning;

// The maximum of a row that sees keys but only scores of -infinity: 0 / 0, as its
// softmax says, where a row that sees nothing (its maximum -infinity) is zero.
constexpr float kAllInf = -std::numeric_limits<float>::max();
__device__ __forceinline__ float inverse_total(float m, float l) {
  return l != 0.0f ? 1.0f / l : m == -__builtin_inff() ? 0.0f : __builtin_nanf("");
}
// Whether a part of a row's keys has sums: those under scores of -infinity alone
// are 0, but 0 * NaN where a value is not finite.
__device__ __forceinline__ bool holds_sums(float m, float l) { return l != 0.0f || m != -__builtin_inff(); }

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
};

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

template <typename T, bool MX, int DP, int WAVES, bool PAGE16, bool ONCE>
__global__ __launch_bounds__(WAVES* kWave, DP * sizeof(T) <= 128 && !MX ? 3 : DP * sizeof(T) <= 256 ? 2 : 1) void attn_rows(AttnDev a) {
  using S = RowsShape<T, MX, DP>;
  constexpr int KT = S::kKeys, NB = S::kBlocks, C = S::kChunk, NV = S::kLoads, AHEAD = S::kAhead;
  constexpr int E = 16 / static_cast<int>(sizeof(T));  // elements of an LDS packet
  __shared__ __align__(16) unsigned char lds[WAVES][2][S::kTileBytes];  // K and V
  __shared__ float2 lds_ml[WAVES][16];
  __shared__ __align__(16) unsigned lds_odd[WAVES][2 * DP];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const int col = lane % 16, g = lane / 16;
  unsigned char* const kl = lds[wave][0];
  unsigned char* const vt = lds[wave][1];

  // Key heads run fastest over the workgroups, so that the XCDs share them out
  // and the row tiles of one head meet in one XCD's L2.
  const unsigned nth = fast_div(blockIdx.x, a.by_kv_heads);
  const int kvh = blockIdx.x - nth * a.kv_heads;
  Item t;
  if (!find_item<16, KT>(a, a.item0 + nth, t)) return;

  const int live = min(16, t.rows - t.row0);
  const int my_token = fast_div(t.row0 + col, a.by_group);  // of the sequence
  const int my_head = kvh * a.group + (t.row0 + col - my_token * a.group);
  const int first_pos = t.pos0 + static_cast<int>(fast_div(t.row0, a.by_group));
  const int last_pos = t.pos0 + static_cast<int>(fast_div(t.row0 + live - 1, a.by_group));
  const KeyTiles kt = t.seq < 0 ? KeyTiles{0, 0, 0, 0} : key_tiles<KT>(a, first_pos, last_pos);
  const int begin = static_cast<int>(static_cast<int64_t>(kt.count) * t.part / t.parts);
  const int end = static_cast<int>(static_cast<int64_t>(kt.count) * (t.part + 1) / t.parts);

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
  // Lane j holds the page of the tile's key j (keys past the end: of the last one).
  const auto look_up = [&](int i) {
    return table[fast_div(min(tile_start(i) + lane % KT, kt.end - 1), a.c.by_page)];
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
  const auto load = [&](Loaded& x, int i, int pages) {
    const int k0 = tile_start(i);
    const RowOffsets<MX> r = row_offsets<T, MX, PAGE16>(a.c, pages, k0 + lane % KT, kt.end);
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
    x.there = static_cast<unsigned>(__ballot(pages >= 0 && pages < a.c.num_pages && lane < KT && k0 + lane < kt.end));
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
  const auto work = [&](Loaded& x, int i) {
    const int k0 = tile_start(i);
    // Whether every live row sees every key of the tile.
    const unsigned here = x.there;
    const bool whole = here == (KT == 32 ? ~0u : 0xffffu) && k0 + KT - 1 <= first_pos &&
                       (a.window <= 0 || k0 > last_pos - a.window || k0 + KT <= a.sinks);
    const unsigned seen = whole ? ~0u : static_cast<unsigned>(keys_seen(here, k0, lo, hi, a.sinks));
    any |= seen;

    // K and V into LDS; rows of V that are not there as zeros.
    wave_fence();
    unsigned odd = 0;  // values that a weight of 0 would not cancel
    if (!whole) {
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        if (!(here >> (n * S::kRowKeys + vkey) & 1)) {
          x.v[n] = u32x4{0, 0, 0, 0};
          x.vcode[n] = kUnitCode;
        }
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
    if (i + AHEAD * WAVES < end) {
      // Loads return in order: the pages of the tile behind it are asked for
      // first, so that using them does not wait for the tile.
      const int now = pages;
      if (i + (AHEAD + 1) * WAVES < end) pages = look_up(i + (AHEAD + 1) * WAVES);
      load(x, i + AHEAD * WAVES, now);
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

  const int first = begin + wave;
#pragma unroll
  for (int n = 0; n < AHEAD; ++n)
    if (first + n * WAVES < end) {
      const int now = n == 0 ? look_up(first) : pages;
      if (first + (n + 1) * WAVES < end) pages = look_up(first + (n + 1) * WAVES);
      load(loaded[n], first + n * WAVES, now);
    }
  for (int i = first; i < end; i += AHEAD * WAVES) {
    work(loaded[0], i);
    if constexpr (AHEAD == 2)
      if (i + WAVES < end) work(loaded[1], i + WAVES);
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
    if (a.max_parts > 1 && t.part == 0 && d == 0) a.row_parts[at] = int2{slot_row, t.parts};
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

// ---- many rows per workgroup ---------------------------------------------------------
// Chunks of a prompt in half types: 32 rows per wavefront, which share each key
// tile through LDS. A tile's loads are issued a whole tile ahead, into registers,
// and go to the other half of LDS after the products of the tile before.
//
// 2048 tokens at the end of 32768 keys, 32 heads of 128 in groups of 4 (1.07 TFLOP
// in bf16): 1251 us, 851 TFLOP/s (1230 to 1272 us over ten runs), where a
// large library product reaches 1255. Counters: matrix cores busy 36% of the cycles, LDS
// 27% without a bank conflict, 97% of the loads from L2. So neither is the bound, but the chain of
// product, maximum, exponentials, product within a wavefront (2.1 us per tile of 64
// keys alone on a CU), and what fills it is other wavefronts: two workgroups
// on a CU, eight wavefronts, at 256 registers each. 64 rows per workgroup: 2142 us.
typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 mfma32(const Eight<__bf16>& a, const Eight<__bf16>& b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(const Eight<_Float16>& a, const Eight<_Float16>& b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Packets of a row of V here: half a wavefront's transposing read takes 64 bytes of
// four keys' rows, which lie on different banks when packets are exchanged in fours.
template <int ROW_BYTES>
__device__ __forceinline__ int lds_packet_v(int key, int p) {
  return key * ROW_BYTES + ((p ^ (ROW_BYTES >= 256 ? (key & 3) << 2 : (key >> 1 & 1) << 2)) << 4);
}

// Four keys' (from `key` on) 16 elements (from d on) transposed by 16 lanes: a lane
// gives the address of 8 bytes and receives its column; then the same 8 keys on.
template <typename T, int ROW_BYTES>
__device__ __forceinline__ Eight<T> read_v(const unsigned char* v, int d, int key, int lane) {
  const int at = d + 4 * (lane % 4), k = key + lane % 16 / 4;
  u32x2 x[2];
#pragma unroll
  for (int n = 0; n < 2; ++n)
    x[n] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4*)(const_cast<unsigned char*>(v) + lds_packet_v<ROW_BYTES>(k + 8 * n, at / 8) + at % 8 * 2)));
  Eight<T> r;
  r.p[0].raw = u32x4{x[0][0], x[0][1], x[1][0], x[1][1]};
  return r;
}

template <typename T, bool MX, int DP, int WAVES, bool PAGE16>
__global__ __launch_bounds__(WAVES* kWave, DP <= 128 ? 2 : 1) void attn_chunk(AttnDev a) {
  constexpr int KT = DP <= 128 ? 64 : 32, R = 32 * WAVES, KB = KT / 32;
  constexpr int ROW = DP * 2, TILE = KT * ROW;       // bytes
  constexpr int C = MX ? 16 : 8;                     // elements of a 16-byte load
  constexpr int LANES = DP / C;                      // lanes across a row
  constexpr int PASS = WAVES * kWave / LANES, NP = KT / PASS;  // keys per pass of the workgroup, passes
  __shared__ __align__(16) unsigned char lds[2][2][TILE];  // buffer, K and V
  __shared__ int lds_odd[2][WAVES];  // of edge tiles: whether infinities or NaN were taken out of V
  __shared__ __align__(16) unsigned lds_masks[2][WAVES][2 * DP];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const int col = lane % 32, h = lane / 32;

  const unsigned nth = fast_div(blockIdx.x, a.by_kv_heads);
  const int kvh = blockIdx.x - nth * a.kv_heads;
  Item t;
  if (!find_item<R, KT>(a, a.item0 + nth, t)) return;

  const int last_row = min(t.row0 + R, t.rows) - 1;
  const auto pos_of = [&](int row) { return t.pos0 + static_cast<int>(fast_div(row, a.by_group)); };
  const KeyTiles kt = t.seq < 0 ? KeyTiles{0, 0, 0, 0} : key_tiles<KT>(a, pos_of(t.row0), pos_of(last_row));
  const int begin = static_cast<int>(static_cast<int64_t>(kt.count) * t.part / t.parts);
  const int end = static_cast<int>(static_cast<int64_t>(kt.count) * (t.part + 1) / t.parts);
  const int first_all = pos_of(t.row0), last_all = pos_of(last_row);

  // The wavefront's rows, and this lane's query.
  const int wrow0 = t.row0 + 32 * wave;
  const bool busy = wrow0 <= last_row;
  const int wfirst = busy ? pos_of(wrow0) : 0, wlast = busy ? pos_of(min(wrow0 + 31, last_row)) : -1;
  const bool row_live = wrow0 + col <= last_row;
  const int my_token = fast_div(wrow0 + col, a.by_group);
  const int my_head = kvh * a.group + (wrow0 + col - my_token * a.group);
  const int hi = row_live ? t.pos0 + my_token : -1;
  const int lo = a.window > 0 ? max(0, max(hi, 0) - a.window + 1) : 0;
  Eight<T> q[DP / 16];
  {
    const int b = a.c.cu ? 0 : t.seq;
    const T* x = static_cast<const T*>(a.q) + b * a.qs[0] + (t.token0 - b * a.c.seq + my_token) * a.qs[1] + my_head * a.qs[2];
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      const int d = 16 * i + 8 * h;
      q[i] = zero_eight<T>();
      if (row_live && d < a.head_dim) q[i] = load_eight<T>(x + d);
      q[i].p[0].raw ^= a.q_sign;
    }
  }

  float m = -__builtin_inff(), l = 0.0f;
  f32x16 o[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[i][r] = 0.0f;

  const int* const table = a.c.table + (t.seq < 0 ? 0 : t.seq * a.c.table_stride);
  const auto tile_start = [&](int i) {
    return i < kt.sink_tiles ? i * KT : kt.low + (i - kt.sink_tiles) * KT;
  };
  // Lane j holds the page of the tile's key j (keys past the end: of the last one).
  const auto look_up = [&](int i) {
    return table[fast_div(min(tile_start(i) + lane % KT, kt.end - 1), a.c.by_page)];
  };
  const auto present = [&](int pg, int i) {
    return __ballot(pg >= 0 && pg < a.c.num_pages && lane < KT && tile_start(i) + lane < kt.end);
  };

  u32x4 kreg[NP], vreg[NP];
  unsigned kcode[NP], vcode[NP];
  constexpr int KPW = kWave / LANES;  // keys of a wavefront's load: at most 16, and they lie inside 16
  constexpr int EB = MX ? 1 : 2;
  const int key0 = threadIdx.x / LANES, part = threadIdx.x % LANES;
  const bool part_in = part * C < a.head_dim;
  const int pd = part_in ? part * C : 0, wkey = lane / LANES;
  const unsigned koff = ((PAGE16 ? wkey * static_cast<unsigned>(a.c.kst[2]) : 0) + pd) * EB;
  const unsigned voff = ((PAGE16 ? wkey * static_cast<unsigned>(a.c.vst[2]) : 0) + pd) * EB;
  const unsigned kcoff = (PAGE16 ? wkey * static_cast<unsigned>(a.c.ksst[2]) : 0) + pd / 32;
  const unsigned vcoff = (PAGE16 ? wkey * static_cast<unsigned>(a.c.vsst[2]) : 0) + pd / 32;
  const HeadPools pools = head_pools<T, MX>(a.c, kvh);
  const auto load_tile = [&](int i, int pages) {
    const RowOffsets<MX> r = row_offsets<T, MX, PAGE16>(a.c, pages, tile_start(i) + lane % KT, kt.end);
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      const int at = n * PASS + wave * KPW;
      kreg[n] = load16<T, MX, false>(pools.k + offset_at<PAGE16>(r.k, at, wkey) + koff);
      if constexpr (MX) kcode[n] = (pools.ks + offset_at<PAGE16>(r.ks, at, wkey))[kcoff];
    }
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      const int at = n * PASS + wave * KPW;
      vreg[n] = load16<T, MX, false>(pools.v + offset_at<PAGE16>(r.v, at, wkey) + voff);
      if constexpr (MX) vcode[n] = (pools.vs + offset_at<PAGE16>(r.vs, at, wkey))[vcoff];
    }
  };
  // A tile that some row of the workgroup does not see whole.
  const auto is_edge = [&](int i, uint64_t here, int first, int last) {
    const int k0 = tile_start(i);
    return here != (KT == 64 ? ~uint64_t(0) : (uint64_t(1) << (KT % 64)) - 1) || k0 + KT - 1 > first ||
           (a.window > 0 && k0 <= last - a.window && k0 + KT > a.sinks);
  };
  // A tile into LDS; returns whether it is an edge for some wavefront, and infinities
  // and NaN were therefore taken out of V for all of them.
  const auto store_tile = [&](int i, int buf, uint64_t here) {
    const bool edge = is_edge(i, here, first_all, last_all);
    unsigned odd = 0;
    if (edge) {
#pragma unroll
      for (int n = 0; n < NP; ++n) {
        if (!(here >> (n * PASS + key0) & 1)) {
          vreg[n] = u32x4{0, 0, 0, 0};
          vcode[n] = kUnitCode;
        }
        odd |= odd_values<T, MX>(vreg[n], MX ? vcode[n] : 0);
      }
      odd = __ballot(odd != 0) != 0;
      if (__builtin_expect(odd, 0)) take_out_odd<T, MX, DP, KPW, NP>(vreg, vcode, lds_masks[buf][wave], lane);
      if (lane == 0) lds_odd[buf][wave] = odd;
    }
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      const int j = n * PASS + key0;
      Eight<T> k[C / 8], v[C / 8];
      if constexpr (MX) {
        const float sk = e8m0_scale(kcode[n]), sv = e8m0_scale(vcode[n]);
        k[0] = from_e4m3<T>(u32x2{kreg[n][0], kreg[n][1]}, sk);
        k[1] = from_e4m3<T>(u32x2{kreg[n][2], kreg[n][3]}, sk);
        v[0] = from_e4m3<T>(u32x2{vreg[n][0], vreg[n][1]}, sv);
        v[1] = from_e4m3<T>(u32x2{vreg[n][2], vreg[n][3]}, sv);
      } else {
        k[0].p[0].raw = kreg[n];
        v[0].p[0].raw = vreg[n];
      }
#pragma unroll
      for (int c = 0; c < C / 8; ++c) {
        if (a.head_dim != DP && !part_in) k[c] = zero_eight<T>();
        const int p = part * (C / 8) + c;
        *reinterpret_cast<u32x4*>(lds[buf][0] + lds_packet_k<ROW>(j, p)) = k[c].p[0].raw;
        *reinterpret_cast<u32x4*>(lds[buf][1] + lds_packet_v<ROW>(j, p)) = v[c].p[0].raw;
      }
    }
    return edge;
  };

  uint64_t here = 0;
  bool taken_out = false;  // of the tile in LDS
  bool any = false;        // the row sees a key
  int pg = 0;
  if (begin < end) {
    pg = look_up(begin);
    here = present(pg, begin);
    load_tile(begin, pg);
    if (begin + 1 < end) pg = look_up(begin + 1);
    taken_out = store_tile(begin, 0, here);
  }
  __syncthreads();
  for (int i = begin; i < end; ++i) {
    const int buf = (i - begin) & 1, k0 = tile_start(i);
    uint64_t next = 0;
    if (i + 1 < end) {
      load_tile(i + 1, pg);
      next = present(pg, i + 1);
      if (i + 2 < end) pg = look_up(i + 2);
    }
    if (busy && k0 <= wlast) {
      const bool edge = is_edge(i, here, wfirst, wlast);
      const unsigned char* const kl = lds[buf][0];
      const unsigned char* const vl = lds[buf][1];
      // S^T: block b holds keys k0 + 32 b + 8 (r / 4) + 4 h + r % 4 of query `col`.
      f32x16 s[KB];
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[b][r] = 0.0f;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d)
#pragma unroll
        for (int b = 0; b < KB; ++b) {
          Eight<T> x;
          x.p[0].raw = *reinterpret_cast<const u32x4*>(kl + lds_packet_k<ROW>(32 * b + col, 2 * d + h));
          s[b] = mfma32(x, q[d], s[b]);
        }
      uint64_t seen = ~uint64_t(0);
      if (edge) {
        seen = keys_seen(here, k0, lo, hi, a.sinks);
#pragma unroll
        for (int b = 0; b < KB; ++b) {
          const unsigned bits = static_cast<unsigned>(seen >> (32 * b)) >> (4 * h);
#pragma unroll
          for (int r = 0; r < 16; ++r) s[b][r] = bits >> (8 * (r / 4) + r % 4) & 1 ? s[b][r] : -__builtin_inff();
        }
      }
      any |= seen != 0;
      float top = -__builtin_inff();
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = __builtin_fmaxf(top, s[b][r]);
      const float mn = __builtin_fmaxf(m, max_of_halves(top));
      const float base = mn == -__builtin_inff() ? 0.0f : mn;
      if (__ballot(mn != m)) {
        const float keep = __builtin_amdgcn_exp2f((m - base) * a.scale_log2);
        l *= keep;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[d][r] *= keep;
        m = mn;
      }
      const float from = Mfma<T>::kShift - base * a.scale_log2;
      Eight<T> p[KT / 16];
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[b][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][r], a.scale_log2, from));
          l += s[b][r];
          p[2 * b + r / 8][r % 8] = from_f32<T>(s[b][r]);
        }
#pragma unroll
      for (int j = 0; j < KT / 16; ++j)
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
          o[d] = mfma32(read_v<T, ROW>(vl, 32 * d + 16 * (lane / 16 % 2), 16 * j + 4 * h, lane), p[j], o[d]);
      // Also by a wavefront whose own rows see the whole tile.
      if (taken_out) {
#pragma nounroll
        for (int w = 0; w < WAVES; ++w) {
          if (__builtin_expect(!__builtin_amdgcn_readfirstlane(lds_odd[buf][w]), 1)) continue;
          unsigned bits = 0;  // the row's keys of wavefront w's loads
#pragma unroll
          for (int n = 0; n < NP; ++n)
            bits |= (static_cast<unsigned>(seen >> (n * PASS + w * KPW)) & ((1u << KPW) - 1)) << (n * KPW);
#pragma unroll
          for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
              const f32x4 x = odd_sums<DP>(lds_masks[buf][w], 32 * d + 2 * r + 4 * h, bits);
#pragma unroll
              for (int k = 0; k < 4; ++k) o[d][r + k] += x[k];
              __builtin_amdgcn_sched_barrier(0);  // rare: not worth registers
            }
        }
      }
    }
    if (i + 1 < end) taken_out = store_tile(i + 1, buf ^ 1, next);
    here = next;
    __syncthreads();
  }

  if (!row_live) return;
  l += __shfl_xor(l, 32);
  m = any && m == -__builtin_inff() ? kAllInf : m * a.scale_log2;
  const int64_t at = int64_t(t.token0 + my_token) * a.q_heads + my_head;
  const int slot_row = ((t.slot + t.part) * a.kv_heads + kvh) * R + 32 * wave + col;
  if (a.max_parts > 1 && t.part == 0 && h == 0) a.row_parts[at] = int2{slot_row, t.parts};
  if (t.parts > 1) {
    if (h == 0) a.part_ml[slot_row] = float2{m, l};
    if (holds_sums(m, l)) {
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
          const int e = 32 * d + 2 * r + 4 * h;
          if (e < a.head_dim)
            *reinterpret_cast<f32x4*>(a.part_o + int64_t(slot_row) * a.head_dim + e) =
                f32x4{o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]};
        }
    }
    return;
  }
  const float inv = inverse_total(m, l);
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int e = 32 * d + 2 * r + 4 * h;
      Pack<T, 4> y;
#pragma unroll
      for (int k = 0; k < 4; ++k) y.e[k] = from_f32<T>(o[d][r + k] * inv);
      if (e < a.head_dim) store_pack<T, 4>(static_cast<T*>(a.out) + at * a.head_dim + e, y);
    }
}

// ---- joining the parts of split key ranges ---------------------------------------
// One wavefront per row whose keys were split: out = sum_s e^(m_s - M) o_s /
// sum_s e^(m_s - M) l_s over its parts, which are `stride` rows apart. Bound by
// latency: LANES lanes hold a part's row, the groups of lanes take every
// (64 / LANES)-th part and eight of them at a time, and are added up at the end; an
// order that depends on nothing but the number of parts. A part without keys
// has no sums and is not read further.
constexpr int kMaxParts = kWave;

template <typename T, int LANES>
__global__ __launch_bounds__(256) void attn_join(const float* __restrict__ part_o, const float2* __restrict__ part_ml,
                                                 const int2* __restrict__ row_parts, T* __restrict__ out, int64_t row0,
                                                 int64_t end, int stride, int64_t part_rows, int head_dim) {
  constexpr int G = kWave / LANES, U = 8;
  const int64_t row = row0 + int64_t(blockIdx.x) * 4 + threadIdx.x / kWave;
  const int lane = threadIdx.x % kWave;
  if (row >= end) return;
  const int2 where = row_parts[row];
  const int n = where.y;
  // Rows that no item covered (a step whose indexes make no sense) hold anything.
  if (n <= 1 || n > kMaxParts || where.x < 0 || where.x + int64_t(n - 1) * stride >= part_rows) return;
  const float2 ml = lane < n ? part_ml[where.x + int64_t(lane) * stride] : float2{-__builtin_inff(), 0.0f};
  float M = ml.x;
#pragma unroll
  for (int k = 1; k < kWave; k *= 2) M = __builtin_fmaxf(M, __shfl_xor(M, k));
  const float w = __builtin_amdgcn_exp2f(ml.x - (M == -__builtin_inff() ? 0.0f : M));
  const uint64_t some = __ballot(holds_sums(ml.x, ml.y));
  const float L = wave_sum(ml.y != 0.0f ? ml.y * w : 0.0f);
  const int d = lane % LANES * 4;
  f32x4 x = {0, 0, 0, 0};
  for (int s0 = 0; s0 < n; s0 += U * G) {  // the same for all lanes, which read each other's weights
    f32x4 y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + lane / LANES + u * G;
      y[u] = f32x4{0, 0, 0, 0};
      if (s < n && (some >> s & 1) && d < head_dim)
        y[u] = *reinterpret_cast<const f32x4*>(part_o + (where.x + int64_t(s) * stride) * head_dim + d);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) x += y[u] * __shfl(w, (s0 + lane / LANES + u * G) % kWave);
  }
#pragma unroll
  for (int k = LANES; k < kWave; k *= 2)
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] += __shfl_xor(x[e], k);
  const float inv = inverse_total(M, L);
  if (lane < LANES && d < head_dim) {
    Pack<T, 4> y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y.e[e] = from_f32<T>(x[e] * inv);
    store_pack<T, 4>(out + row * head_dim + d, y);
  }
}

namespace {

constexpr int kWaves = 4;
constexpr int kChunkRows = 32 * kWaves;

// How a call is cut up: known from what the host knows of it, so that the
// workspace can be sized before the call. The lengths are on the device, so these rules go
// by the table's width, and sequences much shorter than it pay for that: a prompt of 128
// 6.9 us in a table of 128 positions, 13.1 in one of 8192; one token at 128 keys, 32 heads,
// 6.0 and 7.7. Times here are of calls replayed from a graph.
struct Plan {
  bool chunk;         // attn_chunk's row tiles, else attn_rows'
  bool once;          // attn_rows reads (nearly) every key in one workgroup only
  int rows;           // of a row tile
  int64_t row_tiles;  // for one key head, at most
  int64_t items;      // work items wanted for one key head beyond one for each row tile
  int64_t few;        // items for one key head up to which ranges are cut below min_keys
  int max_parts, min_keys;
  int few_keys;       // of a part, where there are few
  int64_t slots;      // row tiles of parts, of all key heads, at most
};

Plan plan(const PagedAttentionArgs& a) {
  const int64_t group = a.q_heads / a.c.kv_heads;
  Plan p{};
  // Rows that share a key head, per sequence (on average in a packed step).
  const int64_t rows = a.c.n_seqs > 0 ? ceil_div(a.c.tokens * group, a.c.n_seqs) : 1;
  // 128 rows share each key tile's way through LDS, 16 do not, but make eight times the
  // workgroups and walk their tiles four at a time. So small launches go to the
  // latter; by the capacity, as the lengths are only known on the device. Measured,
  // heads of 128 in bf16, attn_rows / attn_chunk, by 16-row tiles of all heads times keys:
  // 2^15 (a prompt of 128, 32 heads) 7.5 / 11.4 us, 2^17 (of 256) 9.4 / 15.1,
  // 160 K (16 x 640 keys, 32 rows) 19.5 / 23.4, 2^18 (16384 keys, 32 rows) 36 / 28,
  // 2^19 (a prompt of 512) 25.4 / 22.1, 2^21 (16384 keys, 256 rows) 81 / 43.
  // Up to 16 rows attn_chunk has nothing to share: 8 x 16384 keys 84 / 97.
  const int64_t capacity = a.c.table_width * a.c.page_size;
  const auto row_tiles = [&](int64_t r) { return a.c.cu ? a.c.tokens * group / r + a.c.n_seqs + 1 : a.c.n_seqs * ceil_div(rows, r); };
  constexpr int64_t kSmall = 3 << 16;
  p.chunk = a.dtype != kF32 && rows > 16 && row_tiles(16) * a.c.kv_heads > kSmall / std::max<int64_t>(1, capacity);
  if (a.tuned_kernel > 0) p.chunk = a.dtype != kF32 && a.tuned_kernel == 2;
  p.once = rows <= 16;
  p.rows = p.chunk ? kChunkRows : 16;
  p.row_tiles = row_tiles(p.rows);
  // Two rounds of the two workgroups that a CU holds; attn_chunk's sums of 128 rows
  // are eight times as much to write and join, so one. attn_rows with 512 / 1024 / 2048:
  // 16 x 32768 keys in bf16 347 / 331 / 331 us.
  p.items = ceil_div(a.tuned_items > 0 ? a.tuned_items : p.chunk ? 512 : 1024, a.c.kv_heads);
  // Cutting costs the second kernel, some 4 us. attn_chunk, cut from 256 / from 1024 keys: a prompt
  // of 512 24.6 / 22.1 us, but a ragged packed step, whose longest sequence is the time, 40.7 / 57.9.
  // A packed step may also be that one prompt, and then takes 28.3.
  p.min_keys = a.tuned_min_keys > 0 ? a.tuned_min_keys : p.chunk && !a.c.cu ? 1024 : 256;
  // Few items: one token at 640 keys, 32 heads, in parts of 256 / 64 14.1 / 9.7 us; attn_chunk, 32
  // rows at 2048 keys, 32 heads, in parts of 1024 / 256 60 / 20.4 (such a launch goes to attn_rows: 17.2).
  p.few_keys = std::min(p.min_keys, p.chunk ? 256 : 64);
  // No more than without a window: the workspace is asked for without knowing it.
  const int64_t keys = a.window > 0 ? std::min(capacity, std::min(a.window, capacity) + std::min(a.sinks, capacity)) : capacity;
  p.few = ceil_div(256, a.c.kv_heads);
  p.max_parts = static_cast<int>(std::min<int64_t>(kMaxParts, keys / p.few_keys));
  if (p.max_parts <= 1 || keys <= p.min_keys) {
    p.max_parts = 1;
    p.items = 0;
  } else {
    p.items = std::min(p.items, p.row_tiles * p.max_parts);
    p.slots = p.items * a.c.kv_heads;  // a range that is cut has at most length / L parts
  }
  return p;
}

int64_t workspace_bytes(const PagedAttentionArgs& a, const Plan& p) {
  if (p.max_parts == 1) return 0;
  return p.slots * p.rows * (a.c.head_dim + 2) * static_cast<int64_t>(sizeof(float)) +
         a.c.tokens * a.q_heads * static_cast<int64_t>(sizeof(int2));
}

template <typename T, bool MX, int DP>
hipError_t run(const PagedAttentionArgs& a, hipStream_t stream) {
  const Plan p = plan(a);
  AttnDev d{};
  d.c = paged_dev(a.c);
  d.q = a.q;
  d.out = a.out;
  for (int i = 0; i < 3; ++i) d.qs[i] = a.qs[i];
  d.part_o = static_cast<float*>(a.workspace);
  d.part_ml = reinterpret_cast<float2*>(d.part_o + p.slots * p.rows * a.c.head_dim);
  d.row_parts = reinterpret_cast<int2*>(d.part_ml + p.slots * p.rows);
  d.slots = static_cast<int>(p.slots);
  d.q_heads = static_cast<int>(a.q_heads);
  d.kv_heads = static_cast<int>(a.c.kv_heads);
  d.group = static_cast<int>(a.q_heads / a.c.kv_heads);
  d.head_dim = static_cast<int>(a.c.head_dim);
  const int64_t most = std::numeric_limits<int>::max();
  d.window = static_cast<int>(std::min(a.window, most));
  d.sinks = static_cast<int>(std::min(a.sinks, most));
  d.max_parts = p.max_parts;
  const int tile = p.chunk ? (DP <= 128 ? 64 : 32) : sizeof(T) == 4 ? 16 : 32;
  d.min_tiles = std::max(1, p.min_keys / tile);
  d.few_tiles = std::max(1, p.few_keys / tile);
  d.per_few = 1.0f / static_cast<float>(p.few);
  d.per_item = p.items > 0 ? 1.0f / static_cast<float>(p.items) : 0.0f;
  // Not 0: times it a masked score, -inf, has to stay that.
  d.scale_log2 = std::max(std::fabs(a.scale) * 1.44269504088896340736f, std::numeric_limits<float>::min());
  d.q_sign = a.scale < 0.0f ? (sizeof(T) == 4 ? 0x80000000u : 0x80008000u) : 0u;
  d.by_kv_heads = make_fastdiv(d.kv_heads);
  d.by_group = make_fastdiv(d.group);
  // Rows' offsets inside 16 slots are 32-bit there.
  bool page16 = a.c.page_size % 16 == 0;
  for (const auto* st : {a.c.kst, a.c.vst, a.c.ksst, a.c.vsst}) page16 = page16 && st[2] < (int64_t(1) << 24);
  // Work-items of a launch stay below 2^32.
  const int64_t items = p.row_tiles + p.items, per_launch = std::max<int64_t>(1, (int64_t(1) << 22) / a.c.kv_heads);
  for (int64_t i0 = 0; i0 < items; i0 += per_launch) {
    d.item0 = static_cast<int>(i0);
    const dim3 grid(static_cast<unsigned>(std::min(per_launch, items - i0) * a.c.kv_heads)), block(kWaves * kWave);
    bool launched = false;
    if constexpr (sizeof(T) == 2) {
      if (p.chunk) {
        if (page16) AKO_LAUNCH((attn_chunk<T, MX, DP, kWaves, true>), grid, block, 0, stream, d);
        else AKO_LAUNCH((attn_chunk<T, MX, DP, kWaves, false>), grid, block, 0, stream, d);
        launched = true;
      }
    }
    if (!launched) {
      if (p.once) {
        if (page16) AKO_LAUNCH((attn_rows<T, MX, DP, kWaves, true, true>), grid, block, 0, stream, d);
        else AKO_LAUNCH((attn_rows<T, MX, DP, kWaves, false, true>), grid, block, 0, stream, d);
      } else {
        if (page16) AKO_LAUNCH((attn_rows<T, MX, DP, kWaves, true, false>), grid, block, 0, stream, d);
        else AKO_LAUNCH((attn_rows<T, MX, DP, kWaves, false, false>), grid, block, 0, stream, d);
      }
    }
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  if (p.max_parts == 1) return hipSuccess;
  const int64_t rows = a.c.tokens * a.q_heads;
  constexpr int64_t kJoinRows = int64_t(1) << 24;  // per launch
  for (int64_t r0 = 0; r0 < rows; r0 += kJoinRows) {
    const int64_t n = std::min(kJoinRows, rows - r0);
    AKO_LAUNCH((attn_join<T, DP / 4>), dim3(static_cast<unsigned>(ceil_div(n, 4))), dim3(256), 0, stream, d.part_o, d.part_ml,
               d.row_parts, static_cast<T*>(a.out), r0, r0 + n, d.kv_heads * p.rows, p.slots * p.rows, d.head_dim);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  return hipSuccess;
}

template <typename T, bool MX>
hipError_t by_head_dim(const PagedAttentionArgs& a, hipStream_t stream) {
  if (a.c.head_dim <= 64) return run<T, MX, 64>(a, stream);
  if (a.c.head_dim <= 128) return run<T, MX, 128>(a, stream);
  return run<T, MX, 256>(a, stream);
}

}  // namespace

int64_t paged_attention_workspace(const PagedAttentionArgs& a) { return workspace_bytes(a, plan(a)); }

hipError_t launch_paged_attention(const PagedAttentionArgs& a, hipStream_t stream) {
  switch (a.dtype) {
    case kF32: return a.c.mx ? by_head_dim<float, true>(a, stream) : by_head_dim<float, false>(a, stream);
    case kF16: return a.c.mx ? by_head_dim<_Float16, true>(a, stream) : by_head_dim<_Float16, false>(a, stream);
    case kBF16: return a.c.mx ? by_head_dim<__bf16, true>(a, stream) : by_head_dim<__bf16, false>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace ako

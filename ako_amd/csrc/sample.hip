// A token for each row of logits from a given uniform number, on gfx950.
//
// With m the row's largest logit and T its temperature, token i weighs
//   w_i = e^((x_i - m) / T).
// In descending order of the logits, of equal ones the lowest index first, the
// tokens that stay are the first top_k, of those the shortest run from the front
// that weighs at least top_p of them all, and of those the ones with w_i >= min_p. The
// token drawn is the first, by index, at which the sum of the weights so far passes
// u times the sum of all that stay.
//
// Weights are 64-bit whole numbers, w_i 2^S rounded, S the largest (up to 51) for which
// a row's sum stays below 2^62: sums of whole numbers do not depend on
// their order, so histograms are built with LDS atomics, and the token is the same on every run and
// for every way of dividing the work. A weight is off by 2^-(S+1) of the largest, 2^-46 at
// 131072 tokens; tokens below that count as ruled out, as those with logits of -infinity
// or NaN do.
//
// An element's place in the descending order is a 64-bit number that no other
// has: its logit's bits, in the order of the values, above its index's complement.
// "The k-th" and "where the sum passes P" are the same question for weights 1 and w:
// which element covers a target when the weights are laid end to end. It is answered
// by histograms: bins of the distance to m, then, among the elements of the bin that covers the
// target, bins of their 64-bit numbers, until one element is left.

#include <algorithm>
#include <limits>

#include "common.h"
#include "launch.h"

namespace ako {

struct SampleDev {
  const void* x;
  int64_t stride;
  const float* u;
  // One for each row, or (null) one for all.
  const float* temperatures;
  const int* top_ks;
  const float* top_ps;
  const float* min_ps;
  float temperature, top_p, min_p;
  int top_k;
  int64_t* out;
  int vocab, weight_bits, region_log2;
};

constexpr int kThreads = 1024, kWaves = kThreads / kWave;
constexpr int kBins = 2 * kThreads;  // of a histogram
constexpr int kList = 4096;          // elements held in LDS

// A value's bits in the order of the values; both zeros alike, NaN below all.
__device__ __forceinline__ unsigned sort_bits(float x) {
  const unsigned b = __builtin_bit_cast(unsigned, x + 0.0f);
  return x != x ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_sort_bits(unsigned k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ uint64_t place(float x, int index) {
  return uint64_t(sort_bits(x)) << 32 | (0xffffffffu - static_cast<unsigned>(index));
}
__device__ __forceinline__ float value_at(uint64_t place) { return from_sort_bits(static_cast<unsigned>(place >> 32)); }
__device__ __forceinline__ int index_at(uint64_t place) { return static_cast<int>(0xffffffffu - static_cast<unsigned>(place)); }

// What a row's threads share.
struct SampleLds {
  uint64_t hist[kBins];     // weights by bin of depth, or of place
  uint64_t regions[kBins];  // weights by part of the row
  uint64_t list[kList];
  unsigned count[kBins];
  double pow2[128];         // 2^(j / 128)
  uint64_t wave_sum[kWaves];
  float wave_top[kWaves], wave_low[kWaves];
  int wave_at[kWaves];
  uint64_t lo, hi;          // of the elements of a bin
  unsigned n;               // elements of a bin
  int bin;
  uint64_t before;
};

// The row's own numbers, the same in all threads.
struct SampleRow {
  double top64, per_unit;  // the largest logit, and log2(e) / T
  float top;
  float floor;             // elements from here on weigh something; not -infinity
  float keep;              // elements from here on reach min_p
  float tail;              // elements below here weigh less than 1 - top_p of all together
  float per_bin;           // bins of a unit of logits
  int bits;                // S
  bool flat;               // all that weigh anything weigh the same
};

// 2^(S - t), t log2 units below the largest, rounded to a whole number: 2^(j / 128) from a table
// times 2^z of the rest z, at most 1/256, by its Taylor polynomial of degree 4, off by less than 2^-49.
__device__ __forceinline__ uint64_t weight_of(const SampleLds& l, const SampleRow& r, float x) {
  if (r.flat) return uint64_t(1) << r.bits;
  constexpr double kRound = 0x1.8p45;  // its last bit is 1/128
  constexpr double kLn2 = 0.69314718055994530942;
  const double y = __builtin_fma(static_cast<double>(x) - r.top64, r.per_unit, static_cast<double>(r.bits));
  const double near = y + kRound, z = y - (near - kRound);
  const int j = static_cast<int>(__builtin_bit_cast(uint64_t, near));
  double p = __builtin_fma(z, kLn2 * kLn2 * kLn2 * kLn2 / 24, kLn2 * kLn2 * kLn2 / 6);
  p = __builtin_fma(z, p, kLn2 * kLn2 / 2);
  p = __builtin_fma(z, p, kLn2);
  p = __builtin_fma(z, p, 1.0) * l.pow2[j & 127];  // in [1, 2), or next to it
  const uint64_t scaled = __builtin_bit_cast(uint64_t, p) + (static_cast<uint64_t>(static_cast<unsigned>(j >> 7) << 20) << 32);
  return __builtin_bit_cast(uint64_t, __builtin_bit_cast(double, scaled) + 0x1p52) & 0xfffffffffffffull;
}
__device__ __forceinline__ int bin_of(const SampleRow& r, float x) {
  const float d = x == r.top ? 0.0f : (r.top - x) * r.per_bin;
  return d < static_cast<float>(kBins - 1) ? static_cast<int>(d) : kBins - 1;
}

// The row in packets of 16 bytes: read again for every pass, kRounds of the workgroup's packets
// at a time, or (HELD) kept in LDS after the first.
constexpr int kHeldBytes = 1 << 16;
template <typename T, bool HELD>
struct Row {
  static constexpr int E = 16 / static_cast<int>(sizeof(T)), kRounds = HELD ? 1 : 4;
  using P = Pack<T, E>;
  const T* x;
  int vocab;
  P* held;  // HELD: packet i in place i

  // -infinity behind the end.
  __device__ __forceinline__ P packet(int i) const {
    if (i + E <= vocab) return load_pack<T, E>(x + i);
    P p;
#pragma unroll
    for (int e = 0; e < E; ++e) p.e[e] = i + e < vocab ? x[i + e] : from_f32<T>(-__builtin_inff());
    return p;
  }
  // f(packet, index of its first element); all threads take part in every call. FIRST: of the row's first pass.
  template <bool FIRST = false, typename F>
  __device__ __forceinline__ void each_packet(F f) {
    constexpr int kAtOnce = HELD && FIRST ? 4 : kRounds;
    const int mine = static_cast<int>(threadIdx.x) * E;
#pragma unroll 1
    for (int base = 0; base < vocab; base += kThreads * E * kAtOnce) {
      P p[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int i = base + u * kThreads * E + mine;
        if (HELD && !FIRST) p[u] = held[i / E];
        else p[u] = packet(i);
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int i = base + u * kThreads * E + mine;
        if (base + u * kThreads * E >= vocab) continue;
        if (HELD && FIRST) held[i / E] = p[u];
        f(p[u], i);
        __builtin_amdgcn_sched_barrier(0);  // one packet's work after the other: side by side they would not fit the registers
      }
    }
  }
  // f(element, index).
  template <bool FIRST = false, typename F>
  __device__ __forceinline__ void each(F f) {
    each_packet<FIRST>([&](const P& p, int i) {
#pragma unroll
      for (int e = 0; e < E; ++e) f(to_f32(p.e[e]), i + e);
    });
  }
  __device__ __forceinline__ float at(int i) const { return to_f32(HELD ? held[i / E].e[i % E] : x[i]); }
};

__device__ __forceinline__ void add64(uint64_t* to, uint64_t v) {
  atomicAdd(reinterpret_cast<unsigned long long*>(to), static_cast<unsigned long long>(v));
}
__device__ __forceinline__ void min64(uint64_t* to, uint64_t v) {
  atomicMin(reinterpret_cast<unsigned long long*>(to), static_cast<unsigned long long>(v));
}
__device__ __forceinline__ void max64(uint64_t* to, uint64_t v) {
  atomicMax(reinterpret_cast<unsigned long long*>(to), static_cast<unsigned long long>(v));
}

template <typename W>
__device__ __forceinline__ void clear(W* bins) {
  for (int i = threadIdx.x; i < kBins; i += kThreads) bins[i] = 0;
}

// DPP moves of 32 or 64 bits; lanes without a source take 0.
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned dpp_or_zero(unsigned v) {
  return __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp_or_zero(uint64_t v) {
  return uint64_t(dpp_or_zero<CTRL, ROWS>(static_cast<unsigned>(v >> 32))) << 32 | dpp_or_zero<CTRL, ROWS>(static_cast<unsigned>(v));
}
// The sum of this lane's and all lower lanes' v.
template <typename W>
__device__ __forceinline__ W scan_lanes(W v) {
  v += dpp_or_zero<0x111, 0xF>(v);  // row_shr: 1, 2, 4, 8 inside rows of 16
  v += dpp_or_zero<0x112, 0xF>(v);
  v += dpp_or_zero<0x114, 0xF>(v);
  v += dpp_or_zero<0x118, 0xF>(v);
  v += dpp_or_zero<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
  v += dpp_or_zero<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
  return v;
}
// The sum over the 16 lanes around, in the last of them.
__device__ __forceinline__ uint64_t sum_row16(uint64_t v) {
  v += dpp_or_zero<0x111, 0xF>(v);
  v += dpp_or_zero<0x112, 0xF>(v);
  v += dpp_or_zero<0x114, 0xF>(v);
  return v + dpp_or_zero<0x118, 0xF>(v);
}

__device__ __forceinline__ uint64_t lane64(uint64_t v, int lane) {
  return uint64_t(static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane))) << 32 |
         static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
}

// The bin in which the sum of the bins from the front passes `target` (l.bin, with l.before
// the sum before it; -1 where the total does not pass it); returns the total. Barriers on both sides.
template <typename W>
__device__ __forceinline__ uint64_t find_bin(SampleLds& l, const W* bins, uint64_t target) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  __syncthreads();
  const W a = bins[2 * threadIdx.x], b = bins[2 * threadIdx.x + 1];
  const W upto = scan_lanes(static_cast<W>(a + b));
  if (lane == kWave - 1) l.wave_sum[wave] = upto;
  if (threadIdx.x == 0) l.bin = -1;
  __syncthreads();
  uint64_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const uint64_t s = l.wave_sum[w];
    if (w < wave) before += s;
    total += s;
  }
  before += static_cast<W>(upto - a - b);
  if (before <= target && target < before + a + b) {
    const bool second = target >= before + a;
    l.bin = 2 * threadIdx.x + second;
    l.before = before + (second ? a : 0);
  }
  __syncthreads();
  return total;
}

// The element of the list that covers `target` when the weights are laid end to end in descending
// order of place; the target lies inside. weight(place): 0 for those that do not count.
template <typename F>
__device__ __forceinline__ uint64_t find_in_list(SampleLds& l, int n, uint64_t lo, uint64_t hi, uint64_t target, F weight) {
  const int lane = threadIdx.x % kWave;
  if (n <= kWave) {  // one element a lane, every wavefront by itself
    const uint64_t p = lane < n ? l.list[lane] : 0, w = lane < n ? weight(p) : 0;
    uint64_t before = 0;
    for (int j = 0; j < n; ++j) before += lane64(p, j) > p ? lane64(w, j) : 0;
    const uint64_t hit = __ballot(before <= target && target < before + w);
    return hit != 0 ? lane64(p, __builtin_ctzll(hit)) : lo;
  }
  while (lo < hi) {
    const int shift = max(0, 64 - __builtin_clzll(hi - lo) - 11);  // at most kBins bins
    clear(l.hist);
    clear(l.count);
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const uint64_t p = l.list[i], w = p >= lo && p <= hi ? weight(p) : 0;
      if (w != 0) {
        add64(&l.hist[(hi - p) >> shift], w);
        atomicAdd(&l.count[(hi - p) >> shift], 1u);
      }
    }
    find_bin(l, l.hist, target);
    if (l.bin < 0) return lo;  // not reached: the target lies inside
    const bool alone = l.count[l.bin] == 1;
    target -= l.before;
    hi -= uint64_t(l.bin) << shift;
    const uint64_t span = (uint64_t(1) << shift) - 1;
    lo = hi - lo > span ? hi - span : lo;
    if (alone) {
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const uint64_t p = l.list[i];
        if (p >= lo && p <= hi && weight(p) != 0) l.lo = p;
      }
      __syncthreads();
      lo = hi = l.lo;
    }
    __syncthreads();
  }
  return lo;
}

// Starts a collection of elements: l.n counts them, l.lo and l.hi are the least and greatest places.
__device__ __forceinline__ void begin_list(SampleLds& l) {
  __syncthreads();
  if (threadIdx.x == 0) {
    l.n = 0;
    l.lo = ~uint64_t(0);
    l.hi = 0;
  }
  __syncthreads();
}
// Appends this lane's element, if it is one; all lanes take part. What the list has no room for is counted.
__device__ __forceinline__ void append(SampleLds& l, bool mine, float x, int i) {
  const uint64_t all = __ballot(mine);
  if (all == 0) return;
  const int lane = threadIdx.x % kWave, first = __builtin_ctzll(all);
  unsigned at = 0;
  if (lane == first) at = atomicAdd(&l.n, static_cast<unsigned>(__popcll(all)));
  at = __builtin_amdgcn_readlane(at, first);
  if (mine) {
    const uint64_t p = place(x, i);
    at += __popcll(all & ((uint64_t(1) << lane) - 1));
    if (at < kList) l.list[at] = p;
    min64(&l.lo, p);
    max64(&l.hi, p);
  }
}

// u times the total as a whole number below it.
__device__ __forceinline__ uint64_t drawn(float u, uint64_t total) {
  const double want = (u > 0.0f ? static_cast<double>(u) : 0.0) * static_cast<double>(total);
  return want < static_cast<double>(total) ? min(static_cast<uint64_t>(want), total - 1) : total - 1;
}
// The last of the weights' units that top_p leaves.
__device__ __forceinline__ uint64_t last_unit(float top_p, uint64_t total) {
  const double want = ceil(static_cast<double>(top_p > 0.0f ? top_p : 0.0f) * static_cast<double>(total));
  return want >= 1.0 ? (want < static_cast<double>(total) ? static_cast<uint64_t>(want) : total) - 1 : 0;
}

// All that is left to do for a list of up to 64 elements among which are all that may stay, one a
// lane of one wavefront.
__device__ __forceinline__ void draw_small(const SampleLds& l, const SampleRow& r, int n, int top_k, float top_p, float u, int64_t* out) {
  const int lane = threadIdx.x % kWave;
  const uint64_t p = lane < n ? l.list[lane] : 0, w = lane < n ? weight_of(l, r, value_at(p)) : 0;
  int rank = 0;
  uint64_t before = 0;
  for (int j = 0; j < n; ++j) {
    const bool above = lane64(p, j) > p;
    rank += above;
    before += above ? lane64(w, j) : 0;
  }
  bool stays = lane < n && rank < top_k;
  const uint64_t last = __ballot(lane < n && rank == min(top_k, n) - 1);
  const uint64_t total = lane64(before + w, __builtin_ctzll(last | uint64_t(1) << 63));
  if (top_p < 1.0f) stays = stays && before <= last_unit(top_p, total);
  stays = stays && value_at(p) >= r.keep;
  const uint64_t kept = __ballot(stays);
  uint64_t sum = 0, upto = 0;
  for (int j = 0; j < n; ++j) {
    if (!(kept >> j & 1)) continue;
    const uint64_t x = lane64(w, j);
    sum += x;
    upto += static_cast<unsigned>(lane64(p, j)) > static_cast<unsigned>(p) ? x : 0;  // a lower index
  }
  const uint64_t target = drawn(u, sum);
  if (stays && upto <= target && target < upto + w) *out = index_at(p);
}

template <typename T, bool HELD>
__global__ __launch_bounds__(kThreads) void sample_rows(SampleDev a) {
  __shared__ SampleLds l;
  __shared__ __align__(16) unsigned char held_row[HELD ? kHeldBytes : 16];
  const int64_t n = blockIdx.x;
  Row<T, HELD> row;
  row.x = static_cast<const T*>(a.x) + n * a.stride;
  row.vocab = a.vocab;
  row.held = reinterpret_cast<typename Row<T, HELD>::P*>(held_row);
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const float temperature = a.temperatures ? a.temperatures[n] : a.temperature;
  const int top_k = a.top_ks ? a.top_ks[n] : a.top_k;
  const float top_p = a.top_ps ? a.top_ps[n] : a.top_p, min_p = a.min_ps ? a.min_ps[n] : a.min_p, u = a.u[n];
  const bool greedy = !(temperature > 0.0f) || top_k == 1;
  if (threadIdx.x < 128) l.pow2[threadIdx.x] = exp2(threadIdx.x / 128.0);

  // The largest logit, the first that has it, and the least that is not ruled out.
  float top = -__builtin_inff(), low = __builtin_inff();
  int at = a.vocab;
  if (greedy) {
    row.template each<true>([&](float x, int i) {
      if (x > top) {
        top = x;
        at = i;
      }
    });
  } else {
    row.template each<true>([&](float x, int) {
      top = __builtin_fmaxf(top, x);
      low = __builtin_fminf(low, x > -__builtin_inff() ? x : __builtin_inff());
    });
  }
#pragma unroll
  for (int k = 1; k < kWave; k *= 2) {
    const float x = __shfl_xor(top, k), y = __shfl_xor(low, k);
    const int i = __shfl_xor(at, k);
    at = x > top ? i : x == top ? min(at, i) : at;
    top = __builtin_fmaxf(top, x);
    low = __builtin_fminf(low, y);
  }
  if (lane == 0) {
    l.wave_top[wave] = top;
    l.wave_low[wave] = low;
    l.wave_at[wave] = at;
  }
  clear(l.regions);
  clear(l.hist);
  clear(l.count);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float x = l.wave_top[w];
    at = x > top ? l.wave_at[w] : x == top ? min(at, l.wave_at[w]) : at;
    top = __builtin_fmaxf(top, x);
    low = __builtin_fminf(low, l.wave_low[w]);
  }
  if (greedy || !(top > -__builtin_inff())) {
    if (threadIdx.x == 0) a.out[n] = top > -__builtin_inff() ? at : -1;
    return;
  }

  SampleRow r;
  r.top = top;
  r.top64 = static_cast<double>(top);
  r.per_unit = 1.4426950408889634074 / static_cast<double>(temperature);
  r.bits = a.weight_bits;
  r.flat = !(top < __builtin_inff()) || !(r.per_unit > 0.0);
  const auto below_top = [&](double units) {  // the logit so many log2 units down
    return r.flat ? (top < __builtin_inff() ? -std::numeric_limits<float>::max() : top)
                  : __builtin_fmaxf(static_cast<float>(r.top64 - units / r.per_unit), -std::numeric_limits<float>::max());
  };
  r.floor = below_top(r.bits + 1);
  // As many tokens weigh less than 2^-t of the largest each as there are: together less than 1 - top_p for this t.
  r.tail = top_p < 1.0f ? below_top(fmin(64.0, log2(static_cast<double>(a.vocab) / (1.0 - static_cast<double>(fmaxf(top_p, 0.0f)))) + 1.0)) : 0.0f;
  r.keep = -std::numeric_limits<float>::max();
  if (min_p >= 1.0f) {
    r.keep = top;
  } else if (min_p > 0.0f && !r.flat) {
    const double from = r.top64 + log(static_cast<double>(min_p)) * static_cast<double>(temperature);
    r.keep = __builtin_fmaxf(static_cast<float>(from), r.keep);
    if (static_cast<double>(r.keep) < from) r.keep = from_sort_bits(sort_bits(r.keep) + 1);  // the next one up
  }
  const float span = top - __builtin_fmaxf(low, r.floor);
  r.per_bin = span > 0.0f && span < __builtin_inff() ? static_cast<float>(kBins) / span : 0.0f;

  uint64_t least = 0;   // the place of the last element that stays
  bool listed = false;  // whether all that may stay are in the list
  bool summed = false;  // whether l.regions holds the sums of all that stay
  int held = 0;
  const auto in = [&](float x, int i) { return x >= r.floor && place(x, i) >= least; };
  const auto mass = [&](uint64_t p) { return p >= least ? weight_of(l, r, value_at(p)) : 0; };
  const auto one = [&](uint64_t p) { return static_cast<uint64_t>(p >= least); };

  // The element that covers the target, among those of bin l.bin that the list had no room for: bins of their places.
  const auto resolve = [&](uint64_t lo, uint64_t hi, uint64_t target, bool counts) {
    for (;;) {
      const int shift = max(0, 64 - __builtin_clzll(hi - lo) - 11);
      __syncthreads();
      clear(l.hist);
      __syncthreads();
      row.each([&](float x, int i) {
        const uint64_t p = place(x, i);
        if (p >= lo && p <= hi && in(x, i)) add64(&l.hist[(hi - p) >> shift], counts ? 1 : weight_of(l, r, x));
      });
      find_bin(l, l.hist, target);
      if (l.bin < 0) return lo;  // not reached: the target lies inside
      target -= l.before;
      hi -= uint64_t(l.bin) << shift;
      const uint64_t width = (uint64_t(1) << shift) - 1;
      lo = hi - lo > width ? hi - width : lo;
      begin_list(l);
      row.each([&](float x, int i) {
        const uint64_t p = place(x, i);
        append(l, p >= lo && p <= hi && in(x, i), x, i);
      });
      __syncthreads();
      lo = l.lo;
      hi = l.hi;
      const unsigned found = l.n;
      if (found <= kList)
        return counts ? find_in_list(l, static_cast<int>(found), lo, hi, target, one)
                      : find_in_list(l, static_cast<int>(found), lo, hi, target, mass);
    }
  };

  if (top_k > 0) {
    row.each([&](float x, int) {
      if (x >= r.floor) atomicAdd(&l.count[bin_of(r, x)], 1u);
    });
    find_bin(l, l.count, static_cast<uint64_t>(top_k) - 1);
    const int bin = l.bin;
    if (bin >= 0) {
      const uint64_t before = l.before;
      listed = before + l.count[bin] <= kList;
      begin_list(l);
      row.each([&](float x, int i) {
        const int b = bin_of(r, x);
        append(l, x >= r.floor && (listed ? b <= bin : b == bin), x, i);
      });
      __syncthreads();
      held = static_cast<int>(l.n);
      const uint64_t lo = l.lo, hi = l.hi;
      if (listed && held <= kWave) {
        if (wave == 0) draw_small(l, r, held, top_k, top_p, u, a.out + n);
        return;
      }
      const uint64_t target = static_cast<uint64_t>(top_k) - 1 - (listed ? 0 : before);
      least = held <= kList ? find_in_list(l, held, lo, hi, target, one) : resolve(lo, hi, target, true);
    }
    __syncthreads();
    clear(l.hist);
  }

  if (top_p < 1.0f) {
    if (listed) {
      __syncthreads();
      uint64_t lo = ~uint64_t(0), hi = 0;
      if (threadIdx.x == 0) {
        l.lo = lo;
        l.hi = hi;
      }
      __syncthreads();
      for (int i = threadIdx.x; i < held; i += kThreads) {
        const uint64_t p = l.list[i];
        if (p < least) continue;
        add64(&l.hist[i % kBins], mass(p));  // for the total only
        lo = min(lo, p);
        hi = max(hi, p);
      }
      if (hi != 0) {
        min64(&l.lo, lo);
        max64(&l.hi, hi);
      }
      const uint64_t total = find_bin(l, l.hist, 0);
      lo = l.lo;
      hi = l.hi;
      __syncthreads();
      least = find_in_list(l, held, lo, hi, last_unit(top_p, total), mass);
    } else {
      __syncthreads();
      uint64_t rest = 0;
      row.each([&](float x, int i) {
        if (!in(x, i)) return;
        const uint64_t w = weight_of(l, r, x);
        if (x < r.tail) rest += w;
        else add64(&l.hist[bin_of(r, x)], w);
      });
      if (rest != 0) add64(&l.hist[kBins - 1], rest);  // behind the target in any case
      const uint64_t total = find_bin(l, l.hist, 0), target = last_unit(top_p, total);
      find_bin(l, l.hist, target);
      const int bin = l.bin;
      const uint64_t before = l.before;
      // The bin's elements into the list, and those above it, which stay, to their parts of the row.
      begin_list(l);
      row.each_packet([&](const auto& p, int i) {
        uint64_t sum = 0;
#pragma unroll
        for (int e = 0; e < 16 / static_cast<int>(sizeof(T)); ++e) {
          const float x = to_f32(p.e[e]);
          const int b = bin_of(r, x);
          const bool live = x >= r.floor;
          if (live && b < bin && x >= r.keep && place(x, i + e) >= least) sum += weight_of(l, r, x);
          append(l, live && b == bin && place(x, i + e) >= least, x, i + e);
        }
        if (__ballot(sum != 0) == 0) return;
        sum = sum_row16(sum);  // a part of the row is whole runs of 16 lanes' packets
        if (lane % 16 == 15 && sum != 0) add64(&l.regions[i >> a.region_log2], sum);
      });
      __syncthreads();
      const int found = static_cast<int>(l.n);
      const uint64_t lo = l.lo, hi = l.hi;
      if (found <= kList) {
        least = find_in_list(l, found, lo, hi, target - before, mass);
        for (int i = threadIdx.x; i < found; i += kThreads) {
          const uint64_t p = l.list[i];
          if (p >= least && value_at(p) >= r.keep) add64(&l.regions[index_at(p) >> a.region_log2], weight_of(l, r, value_at(p)));
        }
        summed = true;
      } else {
        __syncthreads();
        clear(l.regions);
        least = resolve(lo, hi, target - before, false);
      }
    }
  }

  // By index: the part of the row in which the sum passes the number drawn, then the token.
  const auto stays = [&](float x, int i) { return in(x, i) && x >= r.keep; };
  __syncthreads();
  if (listed) {
    for (int i = threadIdx.x; i < held; i += kThreads) {
      const uint64_t p = l.list[i];
      if (stays(value_at(p), index_at(p))) add64(&l.regions[index_at(p) >> a.region_log2], weight_of(l, r, value_at(p)));
    }
  } else if (!summed) {
    row.each_packet([&](const auto& p, int i) {
      uint64_t sum = 0;
#pragma unroll
      for (int e = 0; e < 16 / static_cast<int>(sizeof(T)); ++e) {
        const float x = to_f32(p.e[e]);
        if (stays(x, i + e)) sum += weight_of(l, r, x);
      }
      sum = sum_row16(sum);
      if (lane % 16 == 15 && sum != 0) add64(&l.regions[i >> a.region_log2], sum);
    });
  }
  const uint64_t total = find_bin(l, l.regions, 0), target = drawn(u, total);
  find_bin(l, l.regions, target);
  const int region = max(l.bin, 0) << a.region_log2;
  const uint64_t rest = target - l.before;
  for (int i = threadIdx.x; i < kBins; i += kThreads) {
    uint64_t w = 0;
    if (i < (1 << a.region_log2) && region + i < a.vocab) {
      const float x = row.at(region + i);
      if (stays(x, region + i)) w = weight_of(l, r, x);
    }
    l.hist[i] = w;
  }
  find_bin(l, l.hist, rest);
  if (threadIdx.x == 0) a.out[n] = region + max(l.bin, 0);
}

namespace {

template <typename T>
void launch_rows(const SampleDev& d, dim3 grid, hipStream_t stream) {
  if (d.vocab * sizeof(T) <= kHeldBytes) AKO_LAUNCH((sample_rows<T, true>), grid, dim3(kThreads), 0, stream, d);
  else AKO_LAUNCH((sample_rows<T, false>), grid, dim3(kThreads), 0, stream, d);
}

}  // namespace

hipError_t launch_sample(const SampleArgs& a, hipStream_t stream) {
  SampleDev d{};
  d.x = a.x;
  d.u = a.u;
  d.temperatures = a.temperatures;
  d.top_ks = a.top_ks;
  d.top_ps = a.top_ps;
  d.min_ps = a.min_ps;
  d.temperature = a.temperature;
  d.top_k = a.top_k;
  d.top_p = a.top_p;
  d.min_p = a.min_p;
  d.vocab = static_cast<int>(a.vocab);
  int log2 = 0;
  while ((int64_t(1) << log2) < a.vocab) ++log2;
  d.weight_bits = std::min(51, 62 - log2);
  d.region_log2 = std::max(7, log2 - 11);  // at most kBins parts, of 16 lanes' packets or more
  d.stride = a.stride;
  constexpr int64_t kRows = int64_t(1) << 21;  // per launch: work-items stay below 2^32
  for (int64_t r = 0; r < a.rows; r += kRows) {
    const dim3 grid(static_cast<unsigned>(std::min(kRows, a.rows - r)));
    d.x = static_cast<const char*>(a.x) + r * a.stride * dtype_bytes(a.dtype);
    d.u = a.u + r;
    d.temperatures = a.temperatures ? a.temperatures + r : nullptr;
    d.top_ks = a.top_ks ? a.top_ks + r : nullptr;
    d.top_ps = a.top_ps ? a.top_ps + r : nullptr;
    d.min_ps = a.min_ps ? a.min_ps + r : nullptr;
    d.out = a.out + r;
    switch (a.dtype) {
      case kF32: launch_rows<float>(d, grid, stream); break;
      case kF16: launch_rows<_Float16>(d, grid, stream); break;
      case kBF16: launch_rows<__bf16>(d, grid, stream); break;
      default: return hipErrorInvalidValue;
    }
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  return hipSuccess;
}

}  // namespace ako

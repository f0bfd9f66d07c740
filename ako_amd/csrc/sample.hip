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
// 131072 tokens, and by 2^-47 of itself; tokens below the former count as ruled out, as those with logits of -infinity
// or NaN do.
//
// An element's place in the descending order is a 64-bit number that no other
// has: its logit's bits, in the order of the values, above its index's complement.
// "The k-th" and "where the sum passes P" are the same question for weights 1 and w:
// which element covers a target when the weights are laid end to end. It is answered
// by histograms: bins of the distance to m, then, among the elements of the bin that covers the
// target, bins of their 64-bit numbers, until one element is left.
//
// 256 x 131072 in 32 bits with settings of each row's own: 138 us; the first pass reads HBM at 5 TB/s (25), the others
// read again what the last-level cache holds, bound by vector arithmetic and its latency. 1 x 32000 in 16 bits with top_k 50:
// 24 us, a chain of passes in one workgroup.

#include <algorithm>
#include <cmath>
#include <limits>

#include "common.h"
#include "launch.h"
#include "row_rounds.h"

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
  // Rows divided over `parts` workgroups of `chunk` tokens (parts 1: not): each row's share of the workspace.
  unsigned char* space;
  int parts, chunk;
  FastDiv by_parts;
  double pow2[128];  // 2^(j / 128)
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

// What the kernels of a divided row leave for the next: what its workgroups found of the largest logit, the
// histogram of the first stage, the sums of the row's parts, and the elements of the bin.
struct SampleFound {
  float top, low;
  int at;
};
constexpr int kMaxParts = 64;
struct SampleSpace {
  uint64_t hist[kBins];
  uint64_t regions[kBins];
  uint64_t list[kList];
  SampleFound found[kMaxParts];
  unsigned n;  // elements of the bin
  unsigned pad[31];
};
__device__ __forceinline__ SampleSpace* space_of(const SampleDev& a, int64_t n) {
  return reinterpret_cast<SampleSpace*>(a.space) + n;
}

// The row's own numbers, the same in all threads.
struct SampleRow {
  double top64, per_unit;  // the largest finite logit, and log2(e) / T (0 where all that count weigh the same)
  float top;
  float floor;             // elements from here on weigh something; not -infinity
  float keep;              // elements from here on reach min_p
  float tail;              // elements below here weigh less than 1 - top_p of all together
  float per_bin;           // bins of a unit of logits
  double bits;             // S
};

// What a row's threads share.
struct SampleLds {
  uint64_t hist[kBins];     // weights by bin of depth, or of place
  uint64_t regions[kBins];  // weights by part of the row
  uint64_t list[kList];
  unsigned count[kBins];    // elements by bin of place
  double pow2[128];         // 2^(j / 128)
  uint64_t wave_sum[kWaves];
  SampleRow row;
  SampleFound found[kWaves];
  uint64_t lo, hi;          // of the elements of a bin
  unsigned n;               // elements of a bin
  int bin;
  uint64_t before;
};

// 2^(S - t), t log2 units below the largest, rounded to a whole number: 2^(j / 128) from a table
// times 2^z of the rest z, at most 1/256, by its Taylor polynomial of degree 4, off by less than 2^-49.
// Meaningless below r.floor.
template <typename Lds>
__device__ __forceinline__ uint64_t weight_of(const Lds& l, const SampleRow& r, float x) {
  constexpr double kRound = 0x1.8p45;  // its last bit is 1/128
  constexpr double kLn2 = 0.69314718055994530942;
  const double down = static_cast<double>(__builtin_fminf(x, std::numeric_limits<float>::max())) - r.top64;
  const double y = __builtin_fma(down, r.per_unit, r.bits);
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

// The row in packets of 16 bytes, read again for every pass or (HELD) kept in LDS after the
// first. What is left behind the last whole packet comes as packets of one element, in a round of its own.
template <typename T, bool HELD, int THREADS = kThreads>
struct Row {
  static constexpr int E = 16 / static_cast<int>(sizeof(T));
  using P = Pack<T, E>;
  const T* x;
  int whole, rest;  // whole packets, elements behind them
  P* held;          // HELD: round k's packets from place k * THREADS on

  __device__ __forceinline__ Row(const T* row, int vocab, P* lds) : x(row), whole(vocab / E), rest(vocab % E), held(lds) {}
  __device__ __forceinline__ int rounds() const { return rounds_of(whole, rest, THREADS); }
  // The index of the first element of this thread's packet.
  __device__ __forceinline__ int index(int round) const {
    return index_in_round<E>(whole, rest, THREADS, round, static_cast<int>(threadIdx.x));
  }
  // -infinity behind the end.
  __device__ __forceinline__ P packet(int round) const {
    P p;
#pragma unroll
    for (int e = 0; e < E; ++e) p.e[e] = from_f32<T>(-__builtin_inff());
    const int i = round * THREADS + static_cast<int>(threadIdx.x);
    if (rest == 0 || round + 1 < rounds()) {
      if (i < whole) p = load_pack<T, E>(x + int64_t(i) * E);
    } else if (static_cast<int>(threadIdx.x) < rest) {
      p.e[0] = x[whole * E + threadIdx.x];
    }
    return p;
  }
  // f(packet, index of its first element); all threads take part in every call. kAtOnce rounds' packets
  // are on their way together.
  template <typename F>
  __device__ __forceinline__ void each_packet(F f) const {
    constexpr int kAtOnce = HELD ? 4 : 16 / E;
    P p[kAtOnce];
    in_groups<kAtOnce, HELD>(rounds(), [&](int u, int k) { p[u] = HELD ? held[k * THREADS + threadIdx.x] : packet(k); },
                             [&](int u, int k) { f(p[u], index(k)); });
  }
  // The same for the first pass, from memory: four rounds at a time.
  template <typename F>
  __device__ __forceinline__ void first_pass(F f) const {
    P p[4];
    in_groups<4, false>(rounds(), [&](int u, int k) { p[u] = packet(k); },
                        [&](int u, int k) {
                          if (HELD) held[k * THREADS + threadIdx.x] = p[u];
#pragma unroll
                          for (int e = 0; e < E; ++e) f(to_f32(p[u].e[e]), index(k) + e);
                        });
  }
  // f(element, index).
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    each_packet([&](const P& p, int i) {
#pragma unroll
      for (int e = 0; e < E; ++e) f(to_f32(p.e[e]), i + e);
    });
  }
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

// A histogram's running sums: this thread's two bins, what comes before them, and the total.
template <typename W>
struct Bins {
  uint64_t before, total;
  W a, b;

  // Barriers before and inside.
  __device__ __forceinline__ Bins(SampleLds& l, const W* bins) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    __syncthreads();
    a = bins[2 * threadIdx.x];
    b = bins[2 * threadIdx.x + 1];
    const W upto = scan_lanes(static_cast<W>(a + b));
    if (lane == kWave - 1) l.wave_sum[wave] = upto;
    if (threadIdx.x == 0) l.bin = -1;
    __syncthreads();
    before = static_cast<W>(upto - a - b);
    total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const uint64_t s = l.wave_sum[w];
      if (w < wave) before += s;
      total += s;
    }
  }
  // The bin in which the sum from the front passes `target`: l.bin, with l.before the sum before it; -1 where
  // the total does not pass it. Once, with a barrier behind.
  __device__ __forceinline__ void find(SampleLds& l, uint64_t target) const {
    if (before <= target && target < before + a + b) {
      const bool second = target >= before + a;
      l.bin = 2 * threadIdx.x + second;
      l.before = before + (second ? a : 0);
    }
    __syncthreads();
  }
};

// One element a lane, the same in every wavefront (0 behind the n-th): how many of the others are greater, and the sum
// of their weights. The wavefronts compare with a sixteenth of the others each.
struct Ranked {
  int rank;
  uint64_t before;
};
__device__ __forceinline__ Ranked rank_small(SampleLds& l, int n, uint64_t p, uint64_t w) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  __syncthreads();
  if (wave == 0) l.count[lane] = l.hist[lane] = 0;
  __syncthreads();
  unsigned rank = 0;
  uint64_t before = 0;
#pragma unroll
  for (int k = 0; k < kWave / kWaves; ++k) {
    const int j = k * kWaves + wave;
    const bool above = j < n && lane64(p, j) > p;
    rank += above;
    before += above ? lane64(w, j) : 0;
  }
  if (rank != 0) {
    atomicAdd(&l.count[lane], rank);
    add64(&l.hist[lane], before);
  }
  __syncthreads();
  return Ranked{static_cast<int>(l.count[lane]), l.hist[lane]};
}

// The element of the list that covers `target` when the weights are laid end to end in descending
// order of place; the target lies inside. weight(place): 0 for those that do not count.
template <typename F>
__device__ __forceinline__ uint64_t find_in_list(SampleLds& l, int n, uint64_t lo, uint64_t hi, uint64_t target, F weight) {
  const int lane = threadIdx.x % kWave;
  if (n <= kWave) {
    const uint64_t p = lane < n ? l.list[lane] : 0, w = lane < n ? weight(p) : 0;
    const uint64_t before = rank_small(l, n, p, w).before;
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
    Bins<uint64_t>(l, l.hist).find(l, target);
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

// All that is left to do for a list of up to 64 elements among which are all that may stay.
__device__ __forceinline__ void draw_small(SampleLds& l, const SampleRow& r, int n, int top_k, float top_p, float u, int64_t* out) {
  const int lane = threadIdx.x % kWave;
  const uint64_t p = lane < n ? l.list[lane] : 0, w = lane < n ? weight_of(l, r, value_at(p)) : 0;
  const Ranked at = rank_small(l, n, p, w);
  bool stays = lane < n && at.rank < top_k;
  if (top_p < 1.0f) {
    const uint64_t last = __ballot(lane < n && at.rank == min(top_k, n) - 1);
    stays = stays && at.before <= last_unit(top_p, lane64(at.before + w, __builtin_ctzll(last | uint64_t(1) << 63)));
  }
  stays = stays && value_at(p) >= r.keep;
  // By index: the greater an index's complement, the earlier.
  const uint64_t mine = stays ? w : 0, total = lane64(scan_lanes(mine), kWave - 1);
  const uint64_t upto = rank_small(l, n, stays ? static_cast<unsigned>(p) : 0, mine).before;
  const uint64_t target = drawn(u, total);
  if (threadIdx.x < kWave && stays && upto <= target && target < upto + w) *out = index_at(p);
}

// A row's settings; values that a tensor should not hold count as the nearest that it may.
struct Settings {
  float temperature, top_p, min_p;
  int top_k;
  bool greedy;
  __device__ __forceinline__ Settings(const SampleDev& a, int64_t n) {
    temperature = a.temperatures ? a.temperatures[n] : a.temperature;
    top_k = a.top_ks ? a.top_ks[n] : a.top_k;
    top_p = a.top_ps ? a.top_ps[n] : a.top_p;
    min_p = a.min_ps ? a.min_ps[n] : a.min_p;
    if (top_k >= a.vocab) top_k = 0;
    greedy = !(temperature > 0.0f) || top_k == 1;
  }
};

__device__ __forceinline__ SampleRow row_of(const SampleDev& a, const Settings& set, float top, float low) {
  constexpr float kMost = std::numeric_limits<float>::max();
  SampleRow r;
  r.top = top;
  r.top64 = static_cast<double>(__builtin_fminf(top, kMost));
  r.per_unit = top < __builtin_inff() ? 1.4426950408889634074 / static_cast<double>(set.temperature) : 0.0;
  r.bits = a.weight_bits;
  const bool flat = !(r.per_unit > 0.0);
  // The logit so many log2 units down: a bound that only has to be the same everywhere.
  const auto below_top = [&](float units) {
    return flat ? (top < __builtin_inff() ? -kMost : top) : __builtin_fmaxf(top - units / static_cast<float>(r.per_unit), -kMost);
  };
  r.floor = below_top(static_cast<float>(a.weight_bits + 1));
  // As many tokens weigh less than 2^-t of the largest each as there are: together less than 1 - top_p for this t.
  r.tail = set.top_p < 1.0f ? below_top(__builtin_fminf(64.0f, __builtin_log2f(static_cast<float>(a.vocab) / (1.0f - __builtin_fmaxf(set.top_p, 0.0f))) + 1.01f)) : 0.0f;
  r.keep = -kMost;
  if (set.min_p >= 1.0f) {
    r.keep = top;
  } else if (set.min_p > 0.0f && !flat) {
    const double from = r.top64 + log(static_cast<double>(set.min_p)) * static_cast<double>(set.temperature);
    r.keep = __builtin_fmaxf(static_cast<float>(from), r.keep);
    if (static_cast<double>(r.keep) < from) r.keep = from_sort_bits(sort_bits(r.keep) + 1);  // the next one up
  }
  const float span = top - __builtin_fmaxf(low, r.floor);
  r.per_bin = span > 0.0f && span < __builtin_inff() ? static_cast<float>(kBins) / span : 0.0f;
  return r;
}

// ---- a row divided over workgroups ---------------------------------------------------
// Three passes over the row, each a kernel, before sample_rows does the rest: the largest logit; the
// histogram of the first stage (top_k's counts, or top_p's weights), or the sums of the row's parts where
// nothing is left out; the elements of the bin, and the sums of what lies above it. A row whose elements do not fit the list is done anew
// by sample_rows alone.
constexpr int kPartThreads = 256;

template <typename T, int THREADS>
__device__ __forceinline__ Row<T, false, THREADS> part_of_row(const SampleDev& a, int64_t n, int start) {
  return Row<T, false, THREADS>(static_cast<const T*>(a.x) + n * a.stride + start, min(a.chunk, a.vocab - start), nullptr);
}

// The largest logit, the first that has it and the least that is not ruled out, with one more logit. By comparisons, which
// no NaN passes: a maximum with a signalling NaN is NaN, and one of 16 bits arrives here as it was.
__device__ __forceinline__ void look_at(SampleFound& f, float x, int i) {
  f.at = x > f.top ? i : f.at;
  f.top = x > f.top ? x : f.top;
  f.low = x < f.low && x > -__builtin_inff() ? x : f.low;
}

// The same over the lanes of a wavefront.
__device__ __forceinline__ void join_found(SampleFound& f) {
#pragma unroll
  for (int k = 1; k < kWave; k *= 2) {
    const float x = __shfl_xor(f.top, k), y = __shfl_xor(f.low, k);
    const int i = __shfl_xor(f.at, k);
    f.at = x > f.top ? i : x == f.top ? min(f.at, i) : f.at;
    f.top = __builtin_fmaxf(f.top, x);
    f.low = __builtin_fminf(f.low, y);
  }
}
__device__ __forceinline__ SampleFound found_in_row(const SampleDev& a, int64_t n) {
  const int lane = threadIdx.x % kWave;
  SampleFound f{-__builtin_inff(), __builtin_inff(), a.vocab};
  if (lane < a.parts) f = space_of(a, n)->found[lane];
  join_found(f);
  return f;
}

template <typename T>
__global__ __launch_bounds__(kPartThreads) void sample_top(SampleDev a) {
  __shared__ SampleFound waves[kPartThreads / kWave];
  const int64_t n = fast_div(blockIdx.x, a.by_parts);
  const int part = blockIdx.x - static_cast<int>(n) * a.parts, start = part * a.chunk;
  SampleSpace* const space = space_of(a, n);
  for (int i = part * kPartThreads + threadIdx.x; i < kBins; i += a.parts * kPartThreads) space->hist[i] = space->regions[i] = 0;
  if (part == 0 && threadIdx.x == 0) space->n = 0;
  SampleFound f{-__builtin_inff(), __builtin_inff(), a.vocab};
  part_of_row<T, kPartThreads>(a, n, start).first_pass([&](float x, int i) {
    look_at(f, x, start + i);
  });
  join_found(f);
  if (threadIdx.x % kWave == 0) waves[threadIdx.x / kWave] = f;
  __syncthreads();
  if (threadIdx.x >= kWave) return;
  f = SampleFound{-__builtin_inff(), __builtin_inff(), a.vocab};
  if (threadIdx.x < kPartThreads / kWave) f = waves[threadIdx.x];
  join_found(f);
  if (threadIdx.x == 0) space->found[part] = f;
}

// What a part's threads share.
struct PartLds {
  uint64_t hist[kBins];
  double pow2[128];
  SampleRow row;
};
// The row's numbers, formed once for the workgroup: in every wavefront they would take as long as the rest.
template <typename Lds>
__device__ __forceinline__ void share_row(Lds& l, const SampleDev& a, const Settings& set, float top, float low) {
  if (threadIdx.x < kWave) {
    const SampleRow r = row_of(a, set, top, low);
    if (threadIdx.x == 0) l.row = r;
  }
}
__device__ __forceinline__ void add_to_row(const uint64_t* bins, uint64_t* row) {
  for (int i = threadIdx.x; i < kBins; i += kPartThreads)
    if (bins[i] != 0) add64(&row[i], bins[i]);
}

template <typename T>
__global__ __launch_bounds__(kPartThreads) void sample_bins(SampleDev a) {
  __shared__ PartLds l;
  const int64_t n = fast_div(blockIdx.x, a.by_parts);
  const int start = (blockIdx.x - static_cast<int>(n) * a.parts) * a.chunk, lane = threadIdx.x % kWave;
  const Settings set(a, n);
  const SampleFound f = found_in_row(a, n);
  if (set.greedy || !(f.top > -__builtin_inff())) return;
  for (int i = threadIdx.x; i < kBins; i += kPartThreads) l.hist[i] = 0;
  if (threadIdx.x < 128) l.pow2[threadIdx.x] = a.pow2[threadIdx.x];
  share_row(l, a, set, f.top, f.low);
  const auto row = part_of_row<T, kPartThreads>(a, n, start);
  __syncthreads();
  const SampleRow r = l.row;
  if (set.top_k > 0) {
    row.each([&](float x, int) {
      if (x >= r.floor) add64(&l.hist[bin_of(r, x)], 1);
    });
  } else if (set.top_p < 1.0f) {
    uint64_t rest = 0;
    row.each([&](float x, int) {
      const uint64_t w = weight_of(l, r, x);
      rest += x >= r.floor && x < r.tail ? w : 0;
      if (x >= r.floor && !(x < r.tail)) add64(&l.hist[bin_of(r, x)], w);
    });
    if (rest != 0) add64(&l.hist[kBins - 1], rest);  // behind the target in any case
  } else {
    row.each_packet([&](const auto& p, int i) {
      uint64_t sum = 0;
#pragma unroll
      for (int e = 0; e < 16 / static_cast<int>(sizeof(T)); ++e) {
        const float x = to_f32(p.e[e]);
        const bool mine = x >= r.floor && x >= r.keep;
        if (__ballot(mine) != 0) sum += mine ? weight_of(l, r, x) : 0;
      }
      if (__ballot(sum != 0) == 0) return;
      sum = sum_row16(sum);  // a part of the row is whole runs of 16 lanes' packets
      if (lane % 16 == 15 && sum != 0) add64(&l.hist[(start + i) >> a.region_log2], sum);
    });
  }
  __syncthreads();
  SampleSpace* const space = space_of(a, n);
  add_to_row(l.hist, set.top_k > 0 || set.top_p < 1.0f ? space->hist : space->regions);
}

template <typename T>
__global__ __launch_bounds__(kPartThreads) void sample_list(SampleDev a) {
  constexpr int PER = kBins / kPartThreads;
  __shared__ PartLds l;
  __shared__ uint64_t wave_sum[kPartThreads / kWave];
  __shared__ int found_bin;
  __shared__ uint64_t found_before, found_in;
  const int64_t n = fast_div(blockIdx.x, a.by_parts);
  const int start = (blockIdx.x - static_cast<int>(n) * a.parts) * a.chunk;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const Settings set(a, n);
  const SampleFound f = found_in_row(a, n);
  const bool counts = set.top_k > 0;
  if (set.greedy || !(f.top > -__builtin_inff()) || !(counts || set.top_p < 1.0f)) return;
  if (threadIdx.x < 128) l.pow2[threadIdx.x] = a.pow2[threadIdx.x];
  share_row(l, a, set, f.top, f.low);
  SampleSpace* const space = space_of(a, n);
  // The bin that covers the target, found by every part of the row.
  uint64_t bins[PER], mine = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    bins[i] = space->hist[threadIdx.x * PER + i];
    mine += bins[i];
    l.hist[i * kPartThreads + threadIdx.x] = 0;
  }
  const uint64_t upto = scan_lanes(mine);
  if (lane == kWave - 1) wave_sum[wave] = upto;
  if (threadIdx.x == 0) found_bin = -1;
  __syncthreads();
  uint64_t before = upto - mine, total = 0;
  for (int w = 0; w < kPartThreads / kWave; ++w) {
    if (w < wave) before += wave_sum[w];
    total += wave_sum[w];
  }
  const uint64_t target = counts ? static_cast<uint64_t>(set.top_k) - 1 : last_unit(set.top_p, total);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (before <= target && target < before + bins[i]) {
      found_bin = threadIdx.x * PER + i;
      found_before = before;
      found_in = bins[i];
    }
    before += bins[i];
  }
  __syncthreads();
  const int bin = found_bin;
  const SampleRow r = l.row;
  if (bin < 0 || (counts && found_before + found_in > kList)) return;  // no more than top_k, or too many for the list
  part_of_row<T, kPartThreads>(a, n, start).each_packet([&](const auto& p, int i) {
    uint64_t sum = 0;
#pragma unroll
    for (int e = 0; e < 16 / static_cast<int>(sizeof(T)); ++e) {
      const float x = to_f32(p.e[e]);
      const int b = bin_of(r, x);
      const bool live = x >= r.floor, take = live && (counts ? b <= bin : b == bin);
      const uint64_t all = __ballot(take);
      if (all != 0) {
        const int first = __builtin_ctzll(all);
        unsigned at = 0;
        if (lane == first) at = atomicAdd(&space->n, static_cast<unsigned>(__popcll(all)));
        at = __builtin_amdgcn_readlane(at, first) + __popcll(all & ((uint64_t(1) << lane) - 1));
        if (take && at < kList) space->list[at] = place(x, start + i + e);
      }
      if (!counts) {
        const bool stays = live && b < bin && x >= r.keep;
        if (__ballot(stays) != 0) sum += stays ? weight_of(l, r, x) : 0;
      }
    }
    if (counts || __ballot(sum != 0) == 0) return;
    sum = sum_row16(sum);
    if (lane % 16 == 15 && sum != 0) add64(&l.hist[(start + i) >> a.region_log2], sum);
  });
  if (counts) return;
  __syncthreads();
  add_to_row(l.hist, space->regions);
}

// SPLIT: the passes of the first stage are done.
template <typename T, bool HELD, bool SPLIT>
__global__ __launch_bounds__(kThreads) void sample_rows(SampleDev a) {
  using R = Row<T, HELD>;
  __shared__ SampleLds l;
  __shared__ typename R::P held_row[HELD ? held_places(kThreads) : 1];  // and the round behind the whole packets
  const int64_t n = blockIdx.x;
  const R row(static_cast<const T*>(a.x) + n * a.stride, a.vocab, held_row);
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const Settings set(a, n);
  const int top_k = set.top_k;
  const float top_p = set.top_p, u = a.u[n];
  if (threadIdx.x < 128) l.pow2[threadIdx.x] = a.pow2[threadIdx.x];

  // The largest logit, the first that has it, and the least that is not ruled out.
  float top = -__builtin_inff(), low = __builtin_inff();
  int at = a.vocab;
  [[maybe_unused]] SampleSpace* const space = SPLIT ? space_of(a, n) : nullptr;
  if constexpr (SPLIT) {
    const SampleFound f = found_in_row(a, n);
    top = f.top;
    low = f.low;
    at = f.at;
  } else {
    SampleFound f{top, low, at};
    row.first_pass([&](float x, int i) { look_at(f, x, i); });
    join_found(f);
    if (lane == 0) l.found[wave] = f;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float x = l.found[w].top;
      at = x > top ? l.found[w].at : x == top ? min(at, l.found[w].at) : at;
      top = __builtin_fmaxf(top, x);
      low = __builtin_fminf(low, l.found[w].low);
    }
  }
  clear(l.regions);
  clear(l.hist);
  clear(l.count);
  if (set.greedy || !(top > -__builtin_inff())) {
    if (threadIdx.x == 0) a.out[n] = top > -__builtin_inff() ? at : -1;
    return;
  }

  share_row(l, a, set, top, low);
  __syncthreads();
  const SampleRow r = l.row;

  // The last element that stays, and its value and index.
  uint64_t least = 0;
  float least_x = -__builtin_inff();
  int least_i = 0;
  bool listed = false;  // whether all that may stay are in the list
  bool summed = false;  // whether l.regions holds the sums of all that stay
  int held = 0;         // elements in the list
  bool ready = SPLIT;   // what the other kernels have left is still to be used
  const auto in = [&](float x, int i) { return x >= r.floor && (x > least_x || (x == least_x && i <= least_i)); };

  for (int stage = 0; stage < 2; ++stage) {  // top_k, then top_p
    const bool counts = stage == 0;
    if (counts ? top_k <= 0 : !(top_p < 1.0f)) continue;
    const auto weight = [&](uint64_t p) { return p < least ? 0 : counts ? 1 : weight_of(l, r, value_at(p)); };
    uint64_t target = 0, lo = 0, hi = ~uint64_t(0);
    if (listed) {
      __syncthreads();
      clear(l.hist);
      __syncthreads();
      for (int i = threadIdx.x; i < held; i += kThreads) add64(&l.hist[i % kBins], weight(l.list[i]));  // for the total only
      target = last_unit(top_p, Bins<uint64_t>(l, l.hist).total);
      lo = l.lo;
      hi = l.hi;
      __syncthreads();
    } else {
      int bin;
      if (ready) {
        for (int i = threadIdx.x; i < kBins; i += kThreads) l.hist[i] = space->hist[i];
      } else if (counts) {
        row.each([&](float x, int) {
          if (x >= r.floor) add64(&l.hist[bin_of(r, x)], 1);
        });
      } else {
        uint64_t rest = 0;
        row.each([&](float x, int i) {
          const bool mine = in(x, i);
          const uint64_t w = weight_of(l, r, x);
          rest += mine && x < r.tail ? w : 0;
          if (mine && !(x < r.tail)) add64(&l.hist[bin_of(r, x)], w);
        });
        if (rest != 0) add64(&l.hist[kBins - 1], rest);  // behind the target in any case
      }
      const Bins<uint64_t> bins(l, l.hist);
      target = counts ? static_cast<uint64_t>(top_k) - 1 : last_unit(top_p, bins.total);
      bins.find(l, target);
      bin = l.bin;
      if (bin < 0) {  // no more than top_k
        __syncthreads();
        clear(l.hist);
        __syncthreads();
        ready = false;
        continue;
      }
      const uint64_t before = l.before;
      if (counts) listed = before + l.hist[bin] <= kList;
      if (!(counts && listed)) target -= before;
      // The bin's elements into the list (or all up to it), and those above it, which stay, to their parts of the row.
      for (bool again = false;; again = true) {
        begin_list(l);
        if (ready) {
          ready = false;
          held = static_cast<int>(space->n);
          if (counts ? listed : held <= kList) {
            for (int i = threadIdx.x; i < held; i += kThreads) {
              const uint64_t p = l.list[i] = space->list[i];
              min64(&l.lo, p);
              max64(&l.hi, p);
            }
            if (!counts)
              for (int i = threadIdx.x; i < kBins; i += kThreads) l.regions[i] = space->regions[i];
            summed = !counts;
            __syncthreads();
            lo = l.lo;
            hi = l.hi;
            break;
          }
        }
        row.each_packet([&](const typename R::P& p, int i) {
          uint64_t sum = 0;
#pragma unroll
          for (int e = 0; e < R::E; ++e) {
            const float x = to_f32(p.e[e]);
            const int b = bin_of(r, x);
            const bool live = in(x, i + e);
            append(l, live && (counts && listed ? b <= bin : b == bin) && (!again || (place(x, i + e) >= lo && place(x, i + e) <= hi)), x, i + e);
            if (!counts && !again && __ballot(live && b < bin && x >= r.keep) != 0) sum += live && b < bin && x >= r.keep ? weight_of(l, r, x) : 0;
          }
          if (counts || again || __ballot(sum != 0) == 0) return;
          sum = sum_row16(sum);  // a part of the row is whole runs of 16 lanes' packets
          if (lane % 16 == 15 && sum != 0) add64(&l.regions[i >> a.region_log2], sum);
        });
        __syncthreads();
        held = static_cast<int>(l.n);
        lo = l.lo;
        hi = l.hi;
        if (held <= kList) {
          summed = !counts && !again;
          break;
        }
        // Too many: bins of their places.
        const int shift = max(0, 64 - __builtin_clzll(hi - lo) - 11);
        __syncthreads();
        clear(l.hist);
        __syncthreads();
        row.each([&](float x, int i) {
          const uint64_t p = place(x, i);
          if (in(x, i) && p >= lo && p <= hi) add64(&l.hist[(hi - p) >> shift], counts ? 1 : weight_of(l, r, x));
        });
        Bins<uint64_t>(l, l.hist).find(l, target);
        if (l.bin < 0) break;  // not reached: the target lies inside
        target -= l.before;
        hi -= uint64_t(l.bin) << shift;
        const uint64_t width = (uint64_t(1) << shift) - 1;
        lo = hi - lo > width ? hi - width : lo;
      }
      if (counts && listed && held <= kWave) {
        draw_small(l, r, held, top_k, top_p, u, a.out + n);
        return;
      }
    }
    least = find_in_list(l, min(held, kList), lo, hi, target, weight);
    least_x = value_at(least);
    least_i = index_at(least);
    if (summed) {
      for (int i = threadIdx.x; i < held; i += kThreads) {
        const uint64_t p = l.list[i];
        if (p >= least && value_at(p) >= r.keep) add64(&l.regions[index_at(p) >> a.region_log2], weight_of(l, r, value_at(p)));
      }
    }
    __syncthreads();
    if (counts) clear(l.hist);
    __syncthreads();
  }

  // By index: the part of the row in which the sum passes the number drawn, then the token.
  const auto stays = [&](float x, int i) { return in(x, i) && x >= r.keep; };
  if (!summed) {
    clear(l.regions);
    __syncthreads();
    if (SPLIT && ready) {
      for (int i = threadIdx.x; i < kBins; i += kThreads) l.regions[i] = space->regions[i];
    } else if (listed) {
      for (int i = threadIdx.x; i < held; i += kThreads) {
        const uint64_t p = l.list[i];
        if (stays(value_at(p), index_at(p))) add64(&l.regions[index_at(p) >> a.region_log2], weight_of(l, r, value_at(p)));
      }
    } else {
      row.each_packet([&](const typename R::P& p, int i) {
        uint64_t sum = 0;
#pragma unroll
        for (int e = 0; e < R::E; ++e) {
          const float x = to_f32(p.e[e]);
          const bool mine = stays(x, i + e);
          if (__ballot(mine) != 0) sum += mine ? weight_of(l, r, x) : 0;
        }
        if (__ballot(sum != 0) == 0) return;
        sum = sum_row16(sum);
        if (lane % 16 == 15 && sum != 0) add64(&l.regions[i >> a.region_log2], sum);
      });
    }
  }
  const Bins<uint64_t> parts(l, l.regions);
  const uint64_t target = drawn(u, parts.total);
  parts.find(l, target);
  const int region = max(l.bin, 0) << a.region_log2;
  const uint64_t rest = target - l.before;
  for (int i = threadIdx.x; i < kBins; i += kThreads) {
    uint64_t w = 0;
    if (i < (1 << a.region_log2) && region + i < a.vocab) {
      const float x = to_f32(row.x[region + i]);
      if (stays(x, region + i)) w = weight_of(l, r, x);
    }
    l.hist[i] = w;
  }
  Bins<uint64_t>(l, l.hist).find(l, rest);
  if (threadIdx.x == 0) a.out[n] = region + max(l.bin, 0);
}

namespace {

// Workgroups of a row, and tokens of each: 4096 tokens or more, as many as fill the chip with a few rows. Dividing costs
// launches and a second look at every row, and gains where rows are long and leave compute units idle: rows of more than
// 32768 tokens, one for every 512 tokens of a row at most, and no more than compute units. What the host knows of a call's
// settings has no part in it. It loses where rows fill the chip and all have settings of a short chain: at the border,
// 256 rows of 131072, with top_k 50 and for greedy rows, whose later launches have nothing to do. One workgroup a
// row and divided, in us:
//   tokens            131072, 32 bits                             50000, 16 bits         32000, 32 bits
//   rows              1          64         128        256        1          128        1          64         256
//   no settings      65 / 21    69 / 35    75 / 51    81 / 79    30 / 20    32 / 30    24 / 21    25 / 23    29 / 38
//   top_k 50         69 / 30    75 / 60    83 / 77    91 / 107   34 / 29    36 / 52    27 / 30    28 / 37    32 / 65
//   top_p 0.9       110 / 42   141 / 76   151 / 100  157 / 152   61 / 31    70 / 69    39 / 34    47 / 45    51 / 74
//   greedy           16 / 12    17 / 18    22 / 25    25 / 35     9 / 12    10 / 16    14 / 12     9 / 13    11 / 19
// and 159 / 138 for 256 rows of 131072 with mixed settings, where the undivided call takes as long as its slowest row.
struct Parts {
  int parts, chunk;
};
Parts parts_of(int64_t rows, int64_t vocab) {
  constexpr int64_t kStep = 2048;  // a multiple of the regions
  if (vocab <= 32768 || rows > std::min<int64_t>(256, vocab / 512)) return Parts{1, static_cast<int>(vocab)};
  const int64_t most = std::min<int64_t>(kMaxParts, std::max<int64_t>(1, 2048 / rows));
  const int64_t chunk = std::max<int64_t>(4096, ceil_div(ceil_div(vocab, most), kStep) * kStep);
  return Parts{static_cast<int>(ceil_div(vocab, chunk)), static_cast<int>(chunk)};
}

template <typename T>
hipError_t launch_rows(const SampleDev& d, int64_t rows, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(rows)), block(kThreads);
  if (d.parts > 1) {
    const dim3 parts(static_cast<unsigned>(rows * d.parts)), part_block(kPartThreads);
    AKO_LAUNCH((sample_top<T>), parts, part_block, 0, stream, d);
    AKO_LAUNCH((sample_bins<T>), parts, part_block, 0, stream, d);
    AKO_LAUNCH((sample_list<T>), parts, part_block, 0, stream, d);
    AKO_LAUNCH((sample_rows<T, false, true>), grid, block, 0, stream, d);
  } else if (d.vocab * static_cast<int64_t>(sizeof(T)) <= kHeldBytes) {
    AKO_LAUNCH((sample_rows<T, true, false>), grid, block, 0, stream, d);
  } else {
    AKO_LAUNCH((sample_rows<T, false, false>), grid, block, 0, stream, d);
  }
  return hipGetLastError();
}

}  // namespace

int64_t sample_workspace(int64_t rows, int64_t vocab) {
  return parts_of(rows, vocab).parts > 1 ? rows * static_cast<int64_t>(sizeof(SampleSpace)) : 0;
}

hipError_t launch_sample(const SampleArgs& a, hipStream_t stream) {
  SampleDev d{};
  d.temperature = a.temperature;
  d.top_k = a.top_k;
  d.top_p = a.top_p;
  d.min_p = a.min_p;
  d.vocab = static_cast<int>(a.vocab);
  int log2 = 0;
  while ((int64_t(1) << log2) < a.vocab) ++log2;
  d.weight_bits = std::min(51, 62 - log2);
  d.region_log2 = std::max(7, log2 - 11);  // at most kBins parts, of 16 lanes' packets or more
  for (int j = 0; j < 128; ++j) d.pow2[j] = std::exp2(j / 128.0);
  d.stride = a.stride;
  const Parts p = parts_of(a.rows, a.vocab);
  d.space = static_cast<unsigned char*>(a.workspace);
  d.parts = p.parts;
  d.chunk = p.chunk;
  d.by_parts = make_fastdiv(d.parts);
  constexpr int64_t kRows = int64_t(1) << 21;  // per launch: work-items stay below 2^32
  for (int64_t r = 0; r < a.rows; r += kRows) {
    const int64_t rows = std::min(kRows, a.rows - r);
    d.x = static_cast<const char*>(a.x) + r * a.stride * dtype_bytes(a.dtype);
    d.u = a.u + r;
    d.temperatures = a.temperatures ? a.temperatures + r : nullptr;
    d.top_ks = a.top_ks ? a.top_ks + r : nullptr;
    d.top_ps = a.top_ps ? a.top_ps + r : nullptr;
    d.min_ps = a.min_ps ? a.min_ps + r : nullptr;
    d.out = a.out + r;
    hipError_t err = hipErrorInvalidValue;
    switch (a.dtype) {
      case kF32: err = launch_rows<float>(d, rows, stream); break;
      case kF16: err = launch_rows<_Float16>(d, rows, stream); break;
      case kBF16: err = launch_rows<__bf16>(d, rows, stream); break;
    }
    if (err != hipSuccess) return err;
  }
  return hipSuccess;
}

}  // namespace ako

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
  uint64_t hist[kBins];
  uint64_t list[kList];
  unsigned count[kBins];
  double pow2[128];  // 2^(j / 128)
  uint64_t wave_sum[kWaves];
  float wave_top[kWaves], wave_low[kWaves];
  int wave_at[kWaves];
  uint64_t lo, hi;   // of the elements of a bin
  unsigned n;        // elements of a bin
  int bin;
  unsigned bin_count;
  uint64_t before;
};

// The row's own numbers, the same in all threads.
struct SampleRow {
  double per_unit;  // log2(e) / T
  float top;        // the largest logit
  float per_bin;    // bins of a unit of logits
  float dead;       // log2 units below the largest from which on weights are 0
  int bits;         // S
  double low;       // log2 units that min_p leaves
};

// log2 units that x lies below the row's largest.
__device__ __forceinline__ double depth(const SampleRow& r, float x) {
  return x == r.top ? 0.0 : (static_cast<double>(r.top) - static_cast<double>(x)) * r.per_unit;
}
// 2^(S - t) rounded to a whole number: 2^(j / 128) from a table times e^(z ln 2) of the
// rest z, at most 1/256, by its Taylor polynomial of degree 4, off by less than 2^-49.
__device__ __forceinline__ uint64_t weight_of(const SampleLds& l, const SampleRow& r, double t) {
  constexpr double kRound = 0x1.8p45;  // its last bit is 1/128
  const double y = static_cast<double>(r.bits) - t, near = y + kRound;
  const int j = static_cast<int>(__builtin_bit_cast(uint64_t, near));
  const double z = (y - (near - kRound)) * 0.69314718055994530942;
  double p = __builtin_fma(z, 1.0 / 24, 1.0 / 6);
  p = __builtin_fma(z, p, 0.5);
  p = __builtin_fma(z, p, 1.0);
  p = __builtin_fma(z, p, 1.0);
  const double w = __builtin_ldexp(l.pow2[j & 127] * p, j >> 7);
  return __builtin_bit_cast(uint64_t, w + 0x1p52) & 0xfffffffffffffull;
}
__device__ __forceinline__ bool is_live(const SampleRow& r, float x, double t) { return x > -__builtin_inff() && t < r.dead; }
__device__ __forceinline__ int bin_of(const SampleRow& r, float x) {
  const float d = x == r.top ? 0.0f : (r.top - x) * r.per_bin;
  return d < static_cast<float>(kBins - 1) ? static_cast<int>(d) : kBins - 1;
}

// Every element of the row: f(x, index), -infinity behind the end; all threads take part
// in every call. The packets of kUnroll rounds are loaded before the first is used.
template <typename T, typename F>
__device__ __forceinline__ void each_packet(const T* row, int vocab, F f) {
  constexpr int E = 16 / static_cast<int>(sizeof(T)), kUnroll = 4;
  for (int base = 0; base < vocab; base += kThreads * E * kUnroll) {
    Pack<T, E> p[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int i = base + (u * kThreads + static_cast<int>(threadIdx.x)) * E;
      if (i + E <= vocab) {
        p[u] = load_pack<T, E>(row + i);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) p[u].e[e] = i + e < vocab ? row[i + e] : from_f32<T>(-__builtin_inff());
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int i = base + (u * kThreads + static_cast<int>(threadIdx.x)) * E;
      if (base + u * kThreads * E < vocab) f(p[u], i);
    }
  }
}
template <typename T, typename F>
__device__ __forceinline__ void each(const T* row, int vocab, F f) {
  each_packet(row, vocab, [&](const auto& p, int i) {
#pragma unroll
    for (int e = 0; e < 16 / static_cast<int>(sizeof(T)); ++e) f(to_f32(p.e[e]), i + e);
  });
}

__device__ __forceinline__ void clear_bins(SampleLds& l) {
  for (int i = threadIdx.x; i < kBins; i += kThreads) {
    l.hist[i] = 0;
    l.count[i] = 0;
  }
  __syncthreads();
}

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int by) {
  const unsigned lo = __shfl_up(static_cast<unsigned>(v), by), hi = __shfl_up(static_cast<unsigned>(v >> 32), by);
  return uint64_t(hi) << 32 | lo;
}

// The bin in which the sum of the histogram from the front passes `target` (l.bin, with l.before
// the sum before it and l.bin_count its elements; -1 where the total does not pass it); returns the total.
__device__ __forceinline__ uint64_t find_bin(SampleLds& l, uint64_t target) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  __syncthreads();
  const uint64_t a = l.hist[2 * threadIdx.x], b = l.hist[2 * threadIdx.x + 1];
  uint64_t upto = a + b;
#pragma unroll
  for (int k = 1; k < kWave; k *= 2) {
    const uint64_t x = shfl_up64(upto, k);
    if (lane >= k) upto += x;
  }
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
  before += upto - a - b;
  if (before <= target && target < before + a + b) {
    const bool second = target >= before + a;
    l.bin = 2 * threadIdx.x + second;
    l.before = before + (second ? a : 0);
    l.bin_count = l.count[2 * threadIdx.x + second];
  }
  __syncthreads();
  return total;
}

// The element of the list that covers `target` when the weights are laid end to end in descending
// order of place; the target lies inside. weight(place): 0 for those that do not count.
template <typename W>
__device__ __forceinline__ uint64_t find_in_list(SampleLds& l, int n, uint64_t lo, uint64_t hi, uint64_t target, W weight) {
  while (lo < hi) {
    const int shift = max(0, 64 - __builtin_clzll(hi - lo) - 11);  // at most kBins bins
    clear_bins(l);
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const uint64_t p = l.list[i];
      const uint64_t w = p >= lo && p <= hi ? weight(p) : 0;
      if (w != 0) {
        atomicAdd(reinterpret_cast<unsigned long long*>(&l.hist[(hi - p) >> shift]), static_cast<unsigned long long>(w));
        atomicAdd(&l.count[(hi - p) >> shift], 1u);
      }
    }
    find_bin(l, target);
    if (l.bin < 0) return lo;  // not reached: the target lies inside
    target -= l.before;
    hi -= uint64_t(l.bin) << shift;
    const uint64_t span = (uint64_t(1) << shift) - 1;
    lo = hi - lo > span ? hi - span : lo;
    if (l.bin_count == 1) {
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const uint64_t p = l.list[i];
        if (p >= lo && p <= hi && weight(p) != 0) l.lo = p;
      }
      __syncthreads();
      lo = hi = l.lo;
      __syncthreads();
    } else {
      __syncthreads();
    }
  }
  return lo;
}

// Elements for which take(x, index) holds, into the list as places; l.n counts them all, l.lo and
// l.hi are the least and greatest.
template <typename T, typename F>
__device__ __forceinline__ void collect(SampleLds& l, const T* row, int vocab, F take) {
  if (threadIdx.x == 0) {
    l.n = 0;
    l.lo = ~uint64_t(0);
    l.hi = 0;
  }
  __syncthreads();
  const int lane = threadIdx.x % kWave;
  each(row, vocab, [&](float x, int i) {
    const bool mine = take(x, i);
    const uint64_t all = __ballot(mine);
    if (all == 0) return;
    const int first = __builtin_ctzll(all);
    unsigned at = 0;
    if (lane == first) at = atomicAdd(&l.n, static_cast<unsigned>(__popcll(all)));
    at = __builtin_amdgcn_readlane(at, first);
    if (mine) {
      const uint64_t p = place(x, i);
      at += __popcll(all & ((uint64_t(1) << lane) - 1));
      if (at < kList) l.list[at] = p;
      atomicMin(reinterpret_cast<unsigned long long*>(&l.lo), static_cast<unsigned long long>(p));
      atomicMax(reinterpret_cast<unsigned long long*>(&l.hi), static_cast<unsigned long long>(p));
    }
  });
  __syncthreads();
}

// The sum of the 16 lanes around, in all of them.
template <int CTRL>
__device__ __forceinline__ uint64_t dpp_mov64(uint64_t v) {
  const unsigned lo = __builtin_amdgcn_mov_dpp(static_cast<int>(v), CTRL, 0xF, 0xF, false);
  const unsigned hi = __builtin_amdgcn_mov_dpp(static_cast<int>(v >> 32), CTRL, 0xF, 0xF, false);
  return uint64_t(hi) << 32 | lo;
}
__device__ __forceinline__ uint64_t sum16(uint64_t v) {
  v += dpp_mov64<0xB1>(v);
  v += dpp_mov64<0x4E>(v);
  v += dpp_mov64<0x141>(v);
  return v + dpp_mov64<0x140>(v);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_rows(SampleDev a) {
  __shared__ SampleLds l;
  const int64_t n = blockIdx.x;
  const T* const row = static_cast<const T*>(a.x) + n * a.stride;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const float temperature = a.temperatures ? a.temperatures[n] : a.temperature;
  const int top_k = a.top_ks ? a.top_ks[n] : a.top_k;
  const float top_p = a.top_ps ? a.top_ps[n] : a.top_p, min_p = a.min_ps ? a.min_ps[n] : a.min_p;
  const bool greedy = !(temperature > 0.0f) || top_k == 1;
  if (threadIdx.x < 128) l.pow2[threadIdx.x] = exp2(threadIdx.x / 128.0);

  // The largest logit, the first that has it, and the least that is not ruled out.
  float top = -__builtin_inff(), low = __builtin_inff();
  int at = a.vocab;
  each(row, a.vocab, [&](float x, int i) {
    if (x > top) {
      top = x;
      at = i;
    }
    if (x > -__builtin_inff()) low = __builtin_fminf(low, x);
  });
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
  r.per_unit = 1.4426950408889634074 / static_cast<double>(temperature);
  r.bits = a.weight_bits;
  r.dead = static_cast<float>(r.bits + 1);
  r.low = min_p > 0.0f ? fmax(0.0, -log2(static_cast<double>(min_p))) : __builtin_inf();
  const double reach = r.per_unit > 0 ? r.dead / r.per_unit : __builtin_inf();
  const float span = static_cast<float>(fmin(static_cast<double>(top) - static_cast<double>(low), reach));
  r.per_bin = span > 0.0f && span < __builtin_inff() ? static_cast<float>(kBins) / span : 0.0f;

  uint64_t least = 0;   // the place of the last element that stays
  bool listed = false;  // whether all that stay are in the list
  int held = 0;
  const auto in = [&](float x, int i, double& t) {
    t = depth(r, x);
    return is_live(r, x, t) && place(x, i) >= least;
  };
  const auto mass = [&](uint64_t p) { return p >= least ? weight_of(l, r, depth(r, value_at(p))) : 0; };
  const auto one = [&](uint64_t p) { return static_cast<uint64_t>(p >= least); };

  // The element that covers the target, among those of the histogram's bin l.bin.
  const auto resolve = [&](uint64_t target, bool counts) {
    const int bin = l.bin;
    uint64_t lo = 0, hi = ~uint64_t(0);
    target -= l.before;
    for (;;) {
      collect(l, row, a.vocab, [&](float x, int i) {
        double t;
        const uint64_t p = place(x, i);
        return bin_of(r, x) == bin && p >= lo && p <= hi && in(x, i, t);
      });
      lo = l.lo;
      hi = l.hi;
      const unsigned found = l.n;
      __syncthreads();
      if (found <= kList) {
        return counts ? find_in_list(l, static_cast<int>(found), lo, hi, target, one)
                      : find_in_list(l, static_cast<int>(found), lo, hi, target, mass);
      }
      // Too many for the list: bins of their places.
      const int shift = max(0, 64 - __builtin_clzll(hi - lo) - 11);
      clear_bins(l);
      each(row, a.vocab, [&](float x, int i) {
        double t;
        const uint64_t p = place(x, i);
        if (p < lo || p > hi || !in(x, i, t)) return;
        const uint64_t w = counts ? 1 : weight_of(l, r, t);
        atomicAdd(reinterpret_cast<unsigned long long*>(&l.hist[(hi - p) >> shift]), static_cast<unsigned long long>(w));
      });
      find_bin(l, target);
      if (l.bin < 0) return lo;  // not reached
      target -= l.before;
      hi -= uint64_t(l.bin) << shift;
      const uint64_t width = (uint64_t(1) << shift) - 1;
      lo = hi - lo > width ? hi - width : lo;
      __syncthreads();
    }
  };

  if (top_k > 0) {
    clear_bins(l);
    each(row, a.vocab, [&](float x, int i) {
      double t;
      if (in(x, i, t)) atomicAdd(reinterpret_cast<unsigned long long*>(&l.hist[bin_of(r, x)]), 1ull);
    });
    find_bin(l, static_cast<uint64_t>(top_k) - 1);
    const int bin = l.bin;
    if (bin >= 0) {
      const uint64_t all = l.before + l.hist[bin];
      if (all <= kList) {
        __syncthreads();
        collect(l, row, a.vocab, [&](float x, int i) {
          double t;
          return in(x, i, t) && bin_of(r, x) <= bin;
        });
        listed = true;
        held = static_cast<int>(l.n);
        const uint64_t lo = l.lo, hi = l.hi;
        __syncthreads();
        least = find_in_list(l, held, lo, hi, static_cast<uint64_t>(top_k) - 1, one);
      } else {
        least = resolve(static_cast<uint64_t>(top_k) - 1, true);
      }
    }
  }

  if (top_p < 1.0f) {
    clear_bins(l);
    if (listed) {
      for (int i = threadIdx.x; i < held; i += kThreads) {
        const uint64_t p = l.list[i];
        if (p >= least)
          atomicAdd(reinterpret_cast<unsigned long long*>(&l.hist[bin_of(r, value_at(p))]), static_cast<unsigned long long>(mass(p)));
      }
    } else {
      each(row, a.vocab, [&](float x, int i) {
        double t;
        if (in(x, i, t))
          atomicAdd(reinterpret_cast<unsigned long long*>(&l.hist[bin_of(r, x)]), static_cast<unsigned long long>(weight_of(l, r, t)));
      });
    }
    const uint64_t total = find_bin(l, 0);
    const double want = ceil(static_cast<double>(top_p > 0.0f ? top_p : 0.0f) * static_cast<double>(total));
    const uint64_t target = want >= 1.0 ? (want < static_cast<double>(total) ? static_cast<uint64_t>(want) : total) - 1 : 0;
    find_bin(l, target);
    if (listed) {
      uint64_t lo = ~uint64_t(0), hi = 0;
      if (threadIdx.x == 0) {
        l.lo = lo;
        l.hi = hi;
      }
      __syncthreads();
      for (int i = threadIdx.x; i < held; i += kThreads) {
        lo = min(lo, l.list[i]);
        hi = max(hi, l.list[i]);
      }
      atomicMin(reinterpret_cast<unsigned long long*>(&l.lo), static_cast<unsigned long long>(lo));
      atomicMax(reinterpret_cast<unsigned long long*>(&l.hi), static_cast<unsigned long long>(hi));
      __syncthreads();
      lo = l.lo;
      hi = l.hi;
      __syncthreads();
      least = find_in_list(l, held, lo, hi, target, mass);
    } else {
      least = resolve(target, false);
    }
  }

  // By index: the part of the row in which the sum passes the number drawn, then the token.
  const auto stays = [&](float x, int i, double& t) { return in(x, i, t) && t <= r.low; };
  clear_bins(l);
  if (listed) {
    for (int i = threadIdx.x; i < held; i += kThreads) {
      double t;
      const uint64_t p = l.list[i];
      if (stays(value_at(p), index_at(p), t))
        atomicAdd(reinterpret_cast<unsigned long long*>(&l.hist[index_at(p) >> a.region_log2]),
                  static_cast<unsigned long long>(weight_of(l, r, t)));
    }
  } else {
    each_packet(row, a.vocab, [&](const auto& p, int i) {
      uint64_t sum = 0;
#pragma unroll
      for (int e = 0; e < 16 / static_cast<int>(sizeof(T)); ++e) {
        double t;
        if (stays(to_f32(p.e[e]), i + e, t)) sum += weight_of(l, r, t);
      }
      sum = sum16(sum);  // a part of the row is whole runs of 16 lanes' packets
      if (lane % 16 == 0 && sum != 0)
        atomicAdd(reinterpret_cast<unsigned long long*>(&l.hist[i >> a.region_log2]), static_cast<unsigned long long>(sum));
    });
  }
  const uint64_t total = find_bin(l, 0);
  const float u = a.u[n];
  const double want = (u > 0.0f ? static_cast<double>(u) : 0.0) * static_cast<double>(total);
  const uint64_t target = want < static_cast<double>(total) ? min(static_cast<uint64_t>(want), total - 1) : total - 1;
  find_bin(l, target);
  const int region = max(l.bin, 0) << a.region_log2;
  const uint64_t rest = target - l.before;
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += kThreads) {
    uint64_t w = 0;
    if (i < (1 << a.region_log2) && region + i < a.vocab) {
      const float x = to_f32(row[region + i]);
      double t;
      if (stays(x, region + i, t)) w = weight_of(l, r, t);
    }
    l.hist[i] = w;
  }
  find_bin(l, rest);
  if (threadIdx.x == 0) a.out[n] = region + max(l.bin, 0);
}

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
    const dim3 grid(static_cast<unsigned>(std::min(kRows, a.rows - r))), block(kThreads);
    d.x = static_cast<const char*>(a.x) + r * a.stride * dtype_bytes(a.dtype);
    d.u = a.u + r;
    d.temperatures = a.temperatures ? a.temperatures + r : nullptr;
    d.top_ks = a.top_ks ? a.top_ks + r : nullptr;
    d.top_ps = a.top_ps ? a.top_ps + r : nullptr;
    d.min_ps = a.min_ps ? a.min_ps + r : nullptr;
    d.out = a.out + r;
    switch (a.dtype) {
      case kF32: AKO_LAUNCH((sample_rows<float>), grid, block, 0, stream, d); break;
      case kF16: AKO_LAUNCH((sample_rows<_Float16>), grid, block, 0, stream, d); break;
      case kBF16: AKO_LAUNCH((sample_rows<__bf16>), grid, block, 0, stream, d); break;
      default: return hipErrorInvalidValue;
    }
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  return hipSuccess;
}

}  // namespace ako

// A row of packets walked by a workgroup in rounds, one packet a thread and round, a group of rounds at
// a time so that a group's loads are on their way together. Plain C++: the sampling kernels walk with it, and a CPU test
// the same rounds.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define AKO_ROUNDS __host__ __device__ __attribute__((always_inline)) inline
#else
#define AKO_ROUNDS inline
#endif

namespace ako {

// Rounds of a row of `whole` packets and `rest` elements behind them, which come as packets of one element in a
// round of their own.
AKO_ROUNDS int rounds_of(int whole, int rest, int threads) { return (whole + threads - 1) / threads + (rest > 0); }

// The index of the first element of a thread's packet, of E elements; in the round behind the whole packets that of
// its only one.
template <int E>
AKO_ROUNDS int index_in_round(int whole, int rest, int threads, int round, int thread) {
  const int i = round * threads + thread;
  if (rest == 0 || round + 1 < rounds_of(whole, rest, threads)) return i * E;
  return whole * E + (thread < rest ? thread : 0);
}

// load(u, round) for each round of a group, u its place there, then use(u, round) for each. The last group may be
// short: places without a round are left out, or (AGAIN) load the last round again, which costs rows in LDS less than
// a branch before each load (one row of 32000 in 16 bits with top_k 50: 23.7 against 23.9 us).
template <int GROUP, bool AGAIN, typename Load, typename Use>
AKO_ROUNDS void in_groups(int rounds, Load load, Use use) {
#pragma unroll 1
  for (int k0 = 0; k0 < rounds; k0 += GROUP) {
#pragma unroll
    for (int u = 0; u < GROUP; ++u)
      if (AGAIN) load(u, k0 + u < rounds ? k0 + u : rounds - 1);
      else if (k0 + u < rounds) load(u, k0 + u);
#pragma unroll
    for (int u = 0; u < GROUP; ++u) {
      if (k0 + u >= rounds) break;
      use(u, k0 + u);
    }
  }
}

// Rows of up to kHeldBytes stay in LDS after the first pass: round k's packets of 16 bytes from place k * threads on, in
// an array of held_places, with the round behind the whole packets.
constexpr int kHeldBytes = 1 << 16;
constexpr int held_places(int threads) { return kHeldBytes / 16 + threads; }

}  // namespace ako

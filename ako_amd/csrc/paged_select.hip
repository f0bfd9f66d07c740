// Choosing the blocks of a paged cache that a token attends to, on gfx950.
//
// A block is a page. paged_means: the mean of the keys of every page that a step's
// rows have filled, per key head, in 32 bits. select_scores and select_blocks: for each token row
// and key head, of the blocks up to the token's own, the first and last few, and then those
// whose mean key has the largest product with the sum of the queries that share the
// key head, which is `group` times the mean score of the block's keys over those
// heads. Of equal scores the lowest block comes first.
//
// Scores are formed in 64 bits, on the matrix cores: which of two blocks is the k-th
// hangs on the last bits of their scores. Single rows, by vector arithmetic, add up in another order than several, so
// the choice is the same for every batch and every division of the work but where two scores are closer than some
// 2^-50 of the size of their terms.
//
// 16 rows of 1024 blocks of 8 key heads take 27 us, 64 MB of means, 2.4 TB/s: single rows, by vector
// arithmetic. 2048 rows of 512 blocks take 81: 53 for the scores, on the matrix cores at half their 64-bit
// rate (29 us at 71 TFLOP/s), and 28 for the choice.

#include <algorithm>
#include <limits>

#include "paged.h"
#include "select_rule.h"

namespace ako {

// As token_place, for a token of each lane's own.
__device__ __forceinline__ TokenPlace lane_place(const PagedDev& p, int token) {
  if (p.cu == nullptr) return token_place(p, token);
  int lo = 0, hi = p.n_seqs + 1;  // the last i with cu[i] <= token lies in [lo, hi)
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    if (p.cu[mid] <= token) lo = mid;
    else hi = mid;
  }
  if (lo >= p.n_seqs) return TokenPlace{-1, -1};
  const int first = p.cu[lo], end = p.cu[lo + 1];
  if (token < first || token >= end) return TokenPlace{-1, -1};
  return TokenPlace{lo, max(p.lens[lo], 0) - (end - token)};
}

// ---- means of filled pages ---------------------------------------------------------
struct MeansDev {
  PagedDev c;
  float* means;
  int64_t ms[2];  // page, head strides
  int kv_heads, head_dim, lanes, rows;  // lanes across a row, rows of a wavefront's load
  int token0, tile;                     // token rows of a workgroup
  FastDiv by_kv_heads, by_lanes;
};

// A workgroup looks at `tile` token rows for those at the last slot of their page, and takes
// their pages one after the other: each wavefront a quarter of the slots, a kilobyte per load and
// eight loads in flight, added up in the order of the slots' residues and then of
// the wavefronts. Bound by HBM where pages are many: 69 MB of bfloat16 pages in 17.1 us, 4.0 TB/s (a wavefront
// to a page took 48).
template <typename T, bool MX>
__global__ __launch_bounds__(256) void paged_means(MeansDev a) {
  __shared__ float part[4][kWave][9];  // 9: lanes' rows on different banks
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int tile = fast_div(blockIdx.x, a.by_kv_heads), head = blockIdx.x - tile * a.kv_heads;
  const int token = a.token0 + tile * a.tile + lane;
  // Which of the rows fill a page: lane i holds row i's page.
  int page = -1;
  if (lane < a.tile && token < a.c.tokens) {
    const TokenPlace at = lane_place(a.c, token);
    if (at.seq >= 0 && at.pos >= 0 && at.pos < a.c.capacity) {
      int slot;
      page = page_of(a.c, at.seq, at.pos, slot);
      if (slot != a.c.page_size - 1) page = -1;
    }
  }
  const int row = fast_div(lane, a.by_lanes), e0 = (lane - row * a.lanes) * 8;
  for (uint64_t todo = __ballot(page >= 0); todo != 0; todo &= todo - 1) {  // the same in every wavefront
    const int at = __builtin_amdgcn_readlane(page, __builtin_ctzll(todo));
    float sum[8] = {};
    constexpr int U = 8;  // loads in flight
    for (int s0 = wave * a.rows; s0 < a.c.page_size; s0 += U * 4 * a.rows) {
      Eight<float> x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int s = s0 + u * 4 * a.rows + row;
        x[u] = zero_eight<float>();
        if (row >= a.rows || s >= a.c.page_size) continue;
        const int64_t k = at * a.c.kst[0] + head * a.c.kst[1] + s * a.c.kst[2] + e0;
        if constexpr (MX) {
          const unsigned code = a.c.ks[at * a.c.ksst[0] + head * a.c.ksst[1] + s * a.c.ksst[2] + e0 / 32];
          x[u] = from_e4m3<float>(load_bytes8(static_cast<const uint8_t*>(a.c.k) + k), e8m0_scale(code));
        } else {
          const Eight<T> y = load_eight<T>(static_cast<const T*>(a.c.k) + k);
#pragma unroll
          for (int i = 0; i < 8; ++i) x[u][i] = to_f32(y[i]);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] += x[u][i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) part[wave][lane][i] = sum[i];
    __syncthreads();
    for (int e = threadIdx.x; e < a.head_dim; e += 4 * kWave) {
      float total = 0.0f;
      for (int w = 0; w < 4; ++w)
        for (int r = 0; r < a.rows; ++r) total += part[w][r * a.lanes + e / 8][e % 8];
      a.means[at * a.ms[0] + head * a.ms[1] + e] = total / static_cast<float>(a.c.page_size);
    }
    __syncthreads();
  }
}

// ---- scores ---------------------------------------------------------------------------
struct SelectDev {
  PagedDev c;
  const void* q;
  const float* means;
  int64_t qs[3], ms[2];  // q: batch, token, head; means: page, head
  double* scores;        // [rows of the slice, kv_heads, width]; NaN: no such page
  int* out;
  int kv_heads, group, head_dim;
  int count, first, last, width;
  int token0, end;       // the slice's rows
  int tile, chunk;       // rows of a tile, blocks of a workgroup
  FastDiv by_kv_heads, by_tiles;
};

constexpr int kTileRows = 16;  // token rows of a tile, at most

// The blocks that a token at `pos` may attend to are 0 .. blocks - 1.
__device__ __forceinline__ int blocks_of(const SelectDev& a, int pos) {
  return pos < 0 ? 0 : min(static_cast<int>(fast_div(pos, a.c.by_page)) + 1, a.width);
}
__device__ __forceinline__ int page_at(const SelectDev& a, int seq, int block) {
  const int page = a.c.table[seq * a.c.table_stride + block];
  return page >= 0 && page < a.c.num_pages ? page : -1;
}

typedef double f64x2 __attribute__((ext_vector_type(2)));
typedef double f64x4 __attribute__((ext_vector_type(4)));

// Up to 16 token rows by 16 blocks per wavefront and step. The matrix instruction takes four elements of
// the inner dimension from the four groups of 16 lanes; which four is only a name, so group g
// holds packet 4 i + g of a row in its i-th 16 bytes, and a load takes 64 bytes in a row of each of 16 means. (With a quarter of the row
// in each group a load touched 64 lines, which the L1 did not hold until the eighth: 38 us against 31 for 16 rows of 1024 blocks.) The rows' sums of
// queries stay in registers. Rows of a tile that belong to different sequences are
// done one sequence after the other.
template <typename T, int DP>
__global__ __launch_bounds__(256) void select_scores(SelectDev a) {
  constexpr int Q = DP / 4;  // elements of a row in a lane
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, col = lane % 16, g = lane / 16;
  const int head = blockIdx.x - fast_div(blockIdx.x, a.by_kv_heads) * a.kv_heads;
  const unsigned nth = fast_div(blockIdx.x, a.by_kv_heads);
  const int chunk = fast_div(nth, a.by_tiles);
  const int tile = nth - chunk * ((a.end - a.token0 + a.tile - 1) / a.tile);
  const int row0 = a.token0 + tile * a.tile, token = row0 + col;
  const bool live = col < a.tile && token < a.end;
  TokenPlace at{-1, -1};
  if (live) at = lane_place(a.c, token);
  const int blocks = at.seq < 0 ? 0 : blocks_of(a, at.pos);
  // Rows with no more blocks than are asked for are not scored.
  unsigned todo = static_cast<unsigned>(__ballot(blocks > a.count && blocks > chunk * a.chunk)) & 0xffffu;
  if (todo == 0) return;

  double q[Q];
#pragma unroll
  for (int i = 0; i < Q; ++i) q[i] = 0.0;
  if (todo >> col & 1) {
    const int b = a.c.cu ? 0 : at.seq, s = token - b * a.c.seq;
    const T* x = static_cast<const T*>(a.q) + b * a.qs[0] + s * a.qs[1] + int64_t(head) * a.group * a.qs[2] + 4 * g;
    for (int h = 0; h < a.group; ++h, x += a.qs[2]) {
#pragma unroll
      for (int i = 0; i < Q; i += 4) {
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (4 * i + 4 * g < a.head_dim) load_f32<T, 4>(x + 4 * i, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) q[i + j] += static_cast<double>(v[j]);
      }
    }
  }

  while (todo != 0) {
    const int from = __builtin_ctz(todo), seq = __builtin_amdgcn_readlane(at.seq, from);
    const unsigned rows = static_cast<unsigned>(__ballot(at.seq == seq && (todo >> col & 1))) & 0xffffu;
    todo &= ~rows;
    // Positions ascend, so the sequence's last row has the most blocks.
    const int most = __builtin_amdgcn_readlane(blocks, 31 - __builtin_clz(rows));
    for (int b0 = chunk * a.chunk + wave * 16; b0 < min(most, (chunk + 1) * a.chunk); b0 += 4 * 16) {
      const int block = b0 + col, page = block < most ? page_at(a, seq, block) : -1;
      const float* m = a.means + max(page, 0) * a.ms[0] + head * a.ms[1] + 4 * g;
      float k[Q];
#pragma unroll
      for (int i = 0; i < Q; i += 4) {
        Pack<float, 4> p;
        p.raw = u32x4{0, 0, 0, 0};
        if (page >= 0 && 4 * i + 4 * g < a.head_dim) p = load_pack<float, 4>(m + 4 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) k[i + j] = p.e[j];
      }
      f64x4 s = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < Q; ++i) s = __builtin_amdgcn_mfma_f64_16x16x4f64(q[i], static_cast<double>(k[i]), s, 0, 0, 0);
      if (block < most) {
#pragma unroll
        for (int v = 0; v < 4; ++v) {  // a lane holds column `col` of the rows 4 v + g
          const int r = 4 * v + g;
          if (!(rows >> r & 1)) continue;
          const double x = page < 0 ? __builtin_nan("") : s[v] != s[v] ? -__builtin_inf() : s[v];
          a.scores[(int64_t(row0 + r - a.token0) * a.kv_heads + head) * a.width + block] = x;
        }
      }
    }
  }
}

// ---- the choice ---------------------------------------------------------------------
// Doubles as whole numbers in the same order.
__device__ __forceinline__ int64_t order_of(double x) {
  const int64_t b = __builtin_bit_cast(int64_t, x + 0.0);
  return b ^ (b >> 63 & 0x7fffffffffffffffll);
}
__device__ __forceinline__ double of_order(int64_t k) {
  return __builtin_bit_cast(double, k ^ (k >> 63 & 0x7fffffffffffffffll));
}

// The choice for one row and key head, by one wavefront: the score that parts the `want` largest from
// the rest. First for scores rounded to 32 bits, which keeps their order: the interval between
// the least and the greatest is halved until as many lie above as are wanted. Where that meets
// scores that round alike, the interval of the 64-bit scores is halved, first of values,
// then of their bits, until one value is left, whose lowest blocks are then taken. N: scores
// in a lane's registers, 0 where they are too many and are read again for every step.
// score(b): that of block b, NaN where its page is absent.
template <int N, typename Score>
__device__ __forceinline__ void choose(const SelectDev& a, const TokenPlace& at, int blocks, int* out, Score score) {
  const int lane = threadIdx.x % kWave;
  const bool all = blocks <= a.count;
  // Always taken: below `low` and from `high` on, the token's own block being the last.
  const int own = blocks > 0 ? static_cast<int>(fast_div(at.pos, a.c.by_page)) : 0;
  const int low = min(a.first, blocks), high = max(low, min(blocks, max(0, own - a.last + 1)));
  const auto there = [&](int b) {  // scored blocks that are not there are NaN
    if (all) return page_at(a, at.seq, b) >= 0;
    const double x = score(b);
    return x == x;
  };

  // Scores above `cut` are taken, and of those equal to it the first `equal`; `rough`: 32-bit ones from bar on.
  double cut = -__builtin_inf();
  float bar = 0.0f;
  bool rough = false;
  int equal = std::numeric_limits<int>::max();
  // The number of this row's scores between the blocks that are always taken for which f holds; those of absent pages are NaN.
  constexpr int R = N > 0 ? N : 1;
  float mine[R];
  const auto count = [&](auto f) {
    int n = 0;
    if constexpr (N > 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) n += __popcll(__ballot(f(mine[i])));
    } else {
      for (int b0 = low; b0 < high; b0 += kWave) n += __popcll(__ballot(b0 + lane < high && f(static_cast<float>(score(b0 + lane)))));
    }
    return n;
  };
  const auto count64 = [&](auto f) {
    int n = 0;
    for (int b0 = low; b0 < high; b0 += kWave) n += __popcll(__ballot(b0 + lane < high && f(score(b0 + lane))));
    return n;
  };
  if (!all) {
    float least = __builtin_inff(), most = -__builtin_inff();
    const auto widen = [&](float x) {  // NaN changes neither
      least = __builtin_fminf(least, x);
      most = __builtin_fmaxf(most, x);
    };
    if constexpr (N > 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int b = low + i * kWave + lane;
        mine[i] = b < high ? static_cast<float>(score(b)) : __builtin_nanf("");
        widen(mine[i]);
      }
    } else {
      for (int b = low + lane; b < high; b += kWave) widen(static_cast<float>(score(b)));
    }
#pragma unroll
    for (int k = 1; k < kWave; k *= 2) {
      least = __builtin_fminf(least, __shfl_xor(least, k));
      most = __builtin_fmaxf(most, __shfl_xor(most, k));
    }
    int always = 0;
    for (int b0 = 0; b0 < low; b0 += kWave) always += __popcll(__ballot(b0 + lane < low && there(b0 + lane)));
    for (int b0 = high; b0 < blocks; b0 += kWave) always += __popcll(__ballot(b0 + lane < blocks && there(b0 + lane)));
    const int want = max(0, a.count - always);
    if (want == 0) {
      cut = __builtin_inf();
      equal = 0;
    } else if (count([](float x) { return x == x; }) > want) {
      // At least `want` scores are at or above lo, fewer from hi on (all of them lie below infinity, or rounded to it).
      float lo = least, hi = most;
      while (!rough) {
        bar = lo + (hi - lo) * 0.5f;
        if (!(bar > lo && bar <= hi)) break;
        const int above = count([&](float x) { return x >= bar; });
        if (above == want) rough = true;
        else if (above > want) lo = bar;
        else if (bar == hi) break;
        else hi = bar;
      }
      if (!rough) {
        int64_t first = order_of(-__builtin_inf()), end = order_of(__builtin_inf()) + 1;
        for (int step = 0; static_cast<uint64_t>(end) - static_cast<uint64_t>(first) > 1; ++step) {
          int64_t mid = (first & end) + ((first ^ end) >> 1);  // their mean, without overflow
          if (step == 0 && lo > -__builtin_inff()) mid = order_of(lo);
          if (step == 1 && hi < __builtin_inff()) mid = order_of(hi);
          if (step > 1 && step < 32) {
            const double x = 0.5 * of_order(first) + 0.5 * of_order(end);
            if (x == x) mid = order_of(x);
          }
          if (mid <= first || mid >= end) mid = (first & end) + ((first ^ end) >> 1);
          const double at64 = of_order(mid);
          const int above = count64([&](double x) { return x >= at64; });
          if (above >= want) first = mid;
          else end = mid;
          if (above == want) break;
        }
        cut = of_order(first);
        equal = want - count64([&](double x) { return x > cut; });
      }
    }
  }

  int written = 0, equals = 0;
  const uint64_t below = (uint64_t(1) << lane) - 1;
  const auto emit = [&](int b, bool take) {
    const uint64_t taken = __ballot(take);
    const int to = written + __popcll(taken & below);
    if (take && to < a.count) out[to] = b;
    written += __popcll(taken);
  };
  const auto emit_always = [&](int from, int to) {
    for (int b0 = from; b0 < to; b0 += kWave) emit(b0 + lane, b0 + lane < to && there(b0 + lane));
  };
  if (all) {
    emit_always(0, blocks);
  } else {
    emit_always(0, low);
    if (N > 0 && rough) {
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (low + i * kWave < high) emit(low + i * kWave + lane, mine[i] >= bar);
    } else {
      for (int b0 = low; b0 < high; b0 += kWave) {
        const double x = b0 + lane < high ? score(b0 + lane) : __builtin_nan("");
        const uint64_t ties = __ballot(!rough && x == cut);
        bool take = rough ? static_cast<float>(x) >= bar : x > cut;
        if (!rough && x == cut) take = equals + __popcll(ties & below) < equal;
        equals = min(equals + static_cast<int>(__popcll(ties)), std::numeric_limits<int>::max() / 2);
        emit(b0 + lane, take);
      }
    }
    emit_always(high, blocks);
  }
  for (int i = min(written, a.count) + lane; i < a.count; i += kWave) out[i] = -1;
}

// A wavefront per row and key head, from the scores that select_scores has left.
template <int N>
__global__ __launch_bounds__(256) void select_blocks(SelectDev a) {
  const int64_t item = int64_t(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  if (item >= int64_t(a.end - a.token0) * a.kv_heads) return;
  const int row = fast_div(static_cast<unsigned>(item), a.by_kv_heads);
  const TokenPlace at = token_place(a.c, a.token0 + row);
  const double* const scores = a.scores + item * a.width;
  choose<N>(a, at, at.seq < 0 ? 0 : blocks_of(a, at.pos), a.out + (int64_t(a.token0) * a.kv_heads + item) * a.count,
            [&](int b) { return scores[b]; });
}

// Both in one, where a tile's scores fit in LDS: as many rows and blocks as SCORES allows. The
// rows' sums of queries are formed once for the workgroup and lie in LDS too, pairs of them
// exchanged by the row's number so that 16 rows' lie on different banks. A wavefront's means for the
// next 16 blocks are loaded while it works on these, and their pages one step before.
//
// ONE: a single row, whose products leave the matrix cores' other rows empty: each lane adds up
// its quarter of a block's product by itself.
template <typename T, int DP, int SCORES, int WAVES, bool ONE>
__global__ __launch_bounds__(WAVES* kWave, DP <= 128 ? (SCORES > 8192 ? WAVES / 4 : 4) : 2) void select_tile(SelectDev a) {
  constexpr int Q = DP / 4;
  __shared__ double scores[SCORES];
  __shared__ __align__(16) double sums[(ONE ? 1 : kTileRows) * DP];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), col = lane % 16, g = lane / 16;
  const unsigned tile = fast_div(blockIdx.x, a.by_kv_heads);
  const int head = blockIdx.x - tile * a.kv_heads;
  const int row0 = a.token0 + tile * a.tile, token = row0 + col;
  TokenPlace at{-1, -1};
  if (col < a.tile && token < a.end) at = lane_place(a.c, token);
  const int blocks = at.seq < 0 ? 0 : blocks_of(a, at.pos);
  // Rows with no more blocks than are asked for are not scored.
  unsigned todo = static_cast<unsigned>(__ballot(blocks > a.count)) & 0xffffu;

  if (todo != 0) {
    unsigned rows = 0;   // those of the sequence that is worked on
    int seq = 0, most = 0;
    const auto page_of_tile = [&](int b0) { return b0 + col < most ? page_at(a, seq, b0 + col) : -1; };
    Pack<float, 4> next[Q / 4];
    const auto load = [&](int page) {
      const float* m = a.means + max(page, 0) * a.ms[0] + head * a.ms[1] + 4 * g;
#pragma unroll
      for (int i = 0; i < Q / 4; ++i) {
        next[i].raw = u32x4{0, 0, 0, 0};
        if (page >= 0 && 16 * i + 4 * g < a.head_dim) next[i] = load_pack<float, 4>(m + 16 * i);
      }
    };
    int page = -1, ahead = -1;
    const auto begin = [&](unsigned left) {
      const int from = __builtin_ctz(left);
      seq = __builtin_amdgcn_readlane(at.seq, from);
      rows = static_cast<unsigned>(__ballot(at.seq == seq && (left >> col & 1))) & 0xffffu;
      // Positions ascend, so the sequence's last row has the most blocks.
      most = __builtin_amdgcn_readlane(blocks, 31 - __builtin_clz(rows));
      // Loads return in order: a tile's pages are asked for before the means of the tile before it.
      page = page_of_tile(wave * 16);
      ahead = page_of_tile((wave + WAVES) * 16);
      load(page);
    };
    begin(todo);
    for (int i = threadIdx.x; i < a.tile * (DP / 4); i += WAVES * kWave) {
      const int r = i / (DP / 4), e = i % (DP / 4) * 4;
      double sum[4] = {0.0, 0.0, 0.0, 0.0};
      const int seq = __shfl(at.seq, r);  // rows' places stand in the first lanes of every wavefront
      if ((todo >> r & 1) && e < a.head_dim) {
        const int b = a.c.cu ? 0 : seq, s = row0 + r - b * a.c.seq;
        const T* x = static_cast<const T*>(a.q) + b * a.qs[0] + s * a.qs[1] + int64_t(head) * a.group * a.qs[2] + e;
        for (int h = 0; h < a.group; ++h, x += a.qs[2]) {
          float v[4];
          load_f32<T, 4>(x, v);
#pragma unroll
          for (int j = 0; j < 4; ++j) sum[j] += static_cast<double>(v[j]);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; j += 2) *reinterpret_cast<f64x2*>(sums + r * DP + ((e + j) / 2 ^ r) * 2) = f64x2{sum[j], sum[j + 1]};
    }
    __syncthreads();

    for (;;) {
      for (int b0 = wave * 16; b0 < most; b0 += WAVES * 16) {
        Pack<float, 4> k[Q / 4];
#pragma unroll
        for (int i = 0; i < Q / 4; ++i) k[i] = next[i];
        const bool there = page >= 0;
        page = ahead;
        ahead = page_of_tile(b0 + 2 * WAVES * 16);
        load(page);
        const int block = b0 + col;
        if constexpr (ONE) {
          asm volatile("" ::: "memory");  // the sums stay in LDS: in registers they would take 64 of 128
          double x[4] = {0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < Q; ++i) x[i % 4] = __builtin_fma(sums[i / 4 * 16 + 4 * g + i % 4], static_cast<double>(k[i / 4].e[i % 4]), x[i % 4]);
          double s = (x[0] + x[1]) + (x[2] + x[3]);
          s += __shfl_xor(s, 16);
          s += __shfl_xor(s, 32);
          if (g == 0 && block < most) scores[block] = !there ? __builtin_nan("") : s != s ? -__builtin_inf() : s;
          continue;
        }
        f64x4 s = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < Q; i += 2) {
          f64x2 x = {0.0, 0.0};
          if (!ONE && col < a.tile) x = *reinterpret_cast<const f64x2*>(sums + col * DP + (8 * (i / 4) + 2 * g + i % 4 / 2 ^ col) * 2);
#pragma unroll
          for (int j = 0; j < 2; ++j)
            s = __builtin_amdgcn_mfma_f64_16x16x4f64(x[j], static_cast<double>(k[(i + j) / 4].e[(i + j) % 4]), s, 0, 0, 0);
        }
        if (block < most) {
#pragma unroll
          for (int v = 0; v < 4; ++v) {  // a lane holds column `col` of the rows 4 v + g
            const int r = 4 * v + g;
            if (rows >> r & 1) scores[r * a.width + block] = !there ? __builtin_nan("") : s[v] != s[v] ? -__builtin_inf() : s[v];
          }
        }
      }
      todo &= ~rows;
      if (todo == 0) break;
      begin(todo);
    }
    __syncthreads();
  }

  for (int r = wave; r < a.tile; r += WAVES) {
    if (row0 + r >= a.end) break;
    const TokenPlace mine{__builtin_amdgcn_readlane(at.seq, r), __builtin_amdgcn_readlane(at.pos, r)};
    const int n = __builtin_amdgcn_readlane(blocks, r);
    int* const out = a.out + (int64_t(row0 + r) * a.kv_heads + head) * a.count;
    const auto score = [&](int b) { return scores[r * a.width + b]; };
    if (n <= 4 * kWave) choose<4>(a, mine, n, out, score);
    else if (n <= 8 * kWave) choose<8>(a, mine, n, out, score);
    else if (n <= 16 * kWave) choose<16>(a, mine, n, out, score);
    else choose<0>(a, mine, n, out, score);
  }
}

// Workgroups of 256 of a launch, at most, for a call of many rows.
constexpr int64_t kSlice = slice_groups(256);

hipError_t launch_paged_means(const PagedMeansArgs& a, hipStream_t stream) {
  MeansDev d{};
  d.c = paged_dev(a.c);
  d.means = a.means;
  d.ms[0] = a.ms[0];
  d.ms[1] = a.ms[1];
  d.kv_heads = static_cast<int>(a.c.kv_heads);
  d.head_dim = static_cast<int>(a.c.head_dim);
  d.lanes = d.head_dim / 8;
  d.rows = kWave / d.lanes;
  d.by_kv_heads = make_fastdiv(d.kv_heads);
  d.by_lanes = make_fastdiv(d.lanes);
  // A page's worth of a sequence's rows fills one page; single rows of many sequences may each fill theirs, all at once.
  const int64_t per_seq = ceil_div(a.c.tokens, std::max<int64_t>(1, a.c.n_seqs));
  d.tile = static_cast<int>(std::min<int64_t>(kWave, std::max<int64_t>(4, std::min(per_seq, a.c.page_size))));
  const int64_t slice = std::max<int64_t>(1, kSlice / a.c.kv_heads) * d.tile;
  for (int64_t t = 0; t < a.c.tokens; t += slice) {
    d.token0 = static_cast<int>(t);
    const dim3 grid(static_cast<unsigned>(ceil_div(std::min(slice, a.c.tokens - t), d.tile) * a.c.kv_heads)), block(256);
    if (a.c.mx) {
      AKO_LAUNCH((paged_means<float, true>), grid, block, 0, stream, d);
    } else {
      switch (a.dtype) {
        case kF32: AKO_LAUNCH((paged_means<float, false>), grid, block, 0, stream, d); break;
        case kF16: AKO_LAUNCH((paged_means<_Float16, false>), grid, block, 0, stream, d); break;
        case kBF16: AKO_LAUNCH((paged_means<__bf16, false>), grid, block, 0, stream, d); break;
        default: return hipErrorInvalidValue;
      }
    }
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  return hipSuccess;
}

namespace {

// Token rows of a tile: as many as a sequence has on average, since rows of one sequence share its blocks' means.
int tile_rows(const PagedSelectArgs& a) {
  const int64_t per_seq = ceil_div(a.c.tokens, std::max<int64_t>(1, a.c.n_seqs));
  int tile = 1;
  while (tile < kTileRows && tile < per_seq) tile *= 2;
  return tile;
}

// Whether a tile's scores stay in LDS: one launch then, and no scores in memory. On either side of the border, 8 key heads of 128:
// 2048 rows of 896 / 897 blocks take 172 / 216 us, 512 rows 46 / 100, 16 rows, a single tile, 47 / 23.
constexpr int kFewScores = 8192, kMostScores = 14336;
bool in_lds(const PagedSelectArgs& a) { return tile_rows(a) * a.c.table_width <= kMostScores; }

// Token rows whose scores are held at a time: 64 MiB of them, so that they stay in the last level cache.
int64_t slice_rows(const PagedSelectArgs& a) {
  const int64_t row = a.c.kv_heads * a.c.table_width * static_cast<int64_t>(sizeof(double));
  const int64_t rows = std::max<int64_t>(1, (int64_t(1) << 26) / std::max<int64_t>(1, row) / kTileRows) * kTileRows;
  return std::min(rows, a.c.tokens);
}

template <typename T, int DP>
void launch_tile_dim(const SelectDev& d, bool few, dim3 grid, hipStream_t stream) {
  constexpr int kOneWaves = tile_threads(DP, true) / kWave, kTileWaves = tile_threads(DP, false) / kWave;
  if (d.tile == 1) {
    if (few) AKO_LAUNCH((select_tile<T, DP, kFewScores, kOneWaves, true>), grid, dim3(kOneWaves * kWave), 0, stream, d);
    else AKO_LAUNCH((select_tile<T, DP, kMostScores, kOneWaves, true>), grid, dim3(kOneWaves * kWave), 0, stream, d);
  } else {
    if (few) AKO_LAUNCH((select_tile<T, DP, kFewScores, kTileWaves, false>), grid, dim3(kTileWaves * kWave), 0, stream, d);
    else AKO_LAUNCH((select_tile<T, DP, kMostScores, kTileWaves, false>), grid, dim3(kTileWaves * kWave), 0, stream, d);
  }
}
template <typename T>
void launch_tile(const SelectDev& d, bool few, dim3 grid, hipStream_t stream) {
  if (d.head_dim <= 64) launch_tile_dim<T, 64>(d, few, grid, stream);
  else if (d.head_dim <= 128) launch_tile_dim<T, 128>(d, few, grid, stream);
  else launch_tile_dim<T, 256>(d, few, grid, stream);
}

template <typename T>
void launch_scores(const SelectDev& d, dim3 grid, hipStream_t stream) {
  const dim3 block(256);
  if (d.head_dim <= 64) AKO_LAUNCH((select_scores<T, 64>), grid, block, 0, stream, d);
  else if (d.head_dim <= 128) AKO_LAUNCH((select_scores<T, 128>), grid, block, 0, stream, d);
  else AKO_LAUNCH((select_scores<T, 256>), grid, block, 0, stream, d);
}

}  // namespace

int64_t paged_select_workspace(const PagedSelectArgs& a) {
  if (a.c.table_width <= a.count || in_lds(a)) return 0;
  return slice_rows(a) * a.c.kv_heads * a.c.table_width * static_cast<int64_t>(sizeof(double));
}

hipError_t launch_paged_select(const PagedSelectArgs& a, hipStream_t stream) {
  SelectDev d{};
  d.c = paged_dev(a.c);
  d.q = a.q;
  d.means = a.means;
  for (int i = 0; i < 3; ++i) d.qs[i] = a.qs[i];
  d.ms[0] = a.ms[0];
  d.ms[1] = a.ms[1];
  d.scores = static_cast<double*>(a.workspace);
  d.out = a.out;
  d.kv_heads = static_cast<int>(a.c.kv_heads);
  d.group = static_cast<int>(a.q_heads / a.c.kv_heads);
  d.head_dim = static_cast<int>(a.c.head_dim);
  d.count = static_cast<int>(a.count);
  d.first = static_cast<int>(std::min<int64_t>(a.first, a.count));
  d.last = static_cast<int>(a.last);
  d.width = a.c.num_pages > 0 ? static_cast<int>(a.c.table_width) : 0;
  d.by_kv_heads = make_fastdiv(d.kv_heads);
  d.tile = tile_rows(a);
  const bool scored = d.width > a.count;
  if (scored && in_lds(a)) {
    const int64_t rows = tile_slice(a.c.head_dim, d.tile, a.c.kv_heads);
    const bool few = d.tile * a.c.table_width <= kFewScores;
    for (int64_t t = 0; t < a.c.tokens; t += rows) {
      d.token0 = static_cast<int>(t);
      d.end = static_cast<int>(std::min(t + rows, a.c.tokens));
      const dim3 grid(static_cast<unsigned>(ceil_div(d.end - d.token0, d.tile) * a.c.kv_heads));
      switch (a.dtype) {
        case kF32: launch_tile<float>(d, few, grid, stream); break;
        case kF16: launch_tile<_Float16>(d, few, grid, stream); break;
        case kBF16: launch_tile<__bf16>(d, few, grid, stream); break;
        default: return hipErrorInvalidValue;
      }
      const hipError_t err = hipGetLastError();
      if (err != hipSuccess) return err;
    }
    return hipSuccess;
  }
  const int64_t slice = scored ? slice_rows(a) : std::max<int64_t>(1, 4 * kSlice / a.c.kv_heads);
  for (int64_t t = 0; t < a.c.tokens; t += slice) {
    d.token0 = static_cast<int>(t);
    d.end = static_cast<int>(std::min(t + slice, a.c.tokens));
    const int64_t rows = d.end - d.token0, items = rows * a.c.kv_heads;
    if (scored) {
      const int64_t tiles = ceil_div(rows, d.tile), sets = ceil_div(d.width, 64);
      // A workgroup's four wavefronts take 16 blocks each at a time; several times, where there are many.
      const int64_t times = std::min<int64_t>(8, std::max<int64_t>(1, tiles * a.c.kv_heads * sets / 2048));
      d.chunk = static_cast<int>(64 * times);
      d.by_tiles = make_fastdiv(static_cast<unsigned>(tiles));
      const dim3 grid(static_cast<unsigned>(tiles * a.c.kv_heads * ceil_div(d.width, d.chunk)));
      switch (a.dtype) {
        case kF32: launch_scores<float>(d, grid, stream); break;
        case kF16: launch_scores<_Float16>(d, grid, stream); break;
        case kBF16: launch_scores<__bf16>(d, grid, stream); break;
        default: return hipErrorInvalidValue;
      }
      const hipError_t err = hipGetLastError();
      if (err != hipSuccess) return err;
    }
    const dim3 grid(static_cast<unsigned>(ceil_div(items, 4))), block(256);
    // Up to 14336 scores a tile these come with select_tile; so a wide table here, or few blocks of which all are taken.
    if (d.width <= 16 * kWave) AKO_LAUNCH((select_blocks<16>), grid, block, 0, stream, d);
    else if (d.width <= 64 * kWave) AKO_LAUNCH((select_blocks<64>), grid, block, 0, stream, d);
    else AKO_LAUNCH((select_blocks<0>), grid, block, 0, stream, d);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  return hipSuccess;
}

}  // namespace ako

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

#include "paged_rows.h"

namespace ako {

PagedTuning g_paged_tuning;

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

template <typename T, int LANES>
hipError_t join(const AttnDev& d, int64_t rows, int tile, hipStream_t stream) {
  constexpr int64_t kJoinRows = int64_t(1) << 24;  // per launch
  for (int64_t r0 = 0; r0 < rows; r0 += kJoinRows) {
    const int64_t n = std::min(kJoinRows, rows - r0);
    AKO_LAUNCH((attn_join<T, LANES>), dim3(static_cast<unsigned>(ceil_div(n, 4))), dim3(256), 0, stream, d.part_o, d.part_ml,
               d.row_parts, static_cast<T*>(d.out), r0, r0 + n, d.kv_heads * tile, int64_t(d.slots) * tile, d.head_dim);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  return hipSuccess;
}

template <typename T>
hipError_t join_typed(const AttnDev& d, int64_t rows, int tile, hipStream_t stream) {
  if (d.head_dim <= 64) return join<T, 16>(d, rows, tile, stream);
  if (d.head_dim <= 128) return join<T, 32>(d, rows, tile, stream);
  return join<T, 64>(d, rows, tile, stream);
}

}  // namespace

hipError_t launch_attn_join(const AttnDev& d, int dtype, int64_t rows, int tile, hipStream_t stream) {
  switch (dtype) {
    case kF32: return join_typed<float>(d, rows, tile, stream);
    case kF16: return join_typed<_Float16>(d, rows, tile, stream);
    case kBF16: return join_typed<__bf16>(d, rows, tile, stream);
    default: return hipErrorInvalidValue;
  }
}

namespace {

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

template <typename T, bool MX, int DP>
hipError_t run(const PagedAttentionArgs& a, hipStream_t stream) {
  const Plan p = plan(a);
  AttnDev d = attn_dev<T>(a);
  use_workspace(d, a.workspace, p.slots, p.rows);
  const int64_t most = std::numeric_limits<int>::max();
  d.window = static_cast<int>(std::min(a.window, most));
  d.sinks = static_cast<int>(std::min(a.sinks, most));
  d.max_parts = p.max_parts;
  const int tile = p.chunk ? (DP <= 128 ? 64 : 32) : sizeof(T) == 4 ? 16 : 32;
  d.min_tiles = std::max(1, p.min_keys / tile);
  d.few_tiles = std::max(1, p.few_keys / tile);
  d.per_few = 1.0f / static_cast<float>(p.few);
  d.per_item = p.items > 0 ? 1.0f / static_cast<float>(p.items) : 0.0f;
  const bool page16 = pages_of_16(a.c);
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
        if (page16) AKO_LAUNCH((attn_rows<T, MX, DP, kWaves, true, true, false>), grid, block, 0, stream, d);
        else AKO_LAUNCH((attn_rows<T, MX, DP, kWaves, false, true, false>), grid, block, 0, stream, d);
      } else {
        if (page16) AKO_LAUNCH((attn_rows<T, MX, DP, kWaves, true, false, false>), grid, block, 0, stream, d);
        else AKO_LAUNCH((attn_rows<T, MX, DP, kWaves, false, false, false>), grid, block, 0, stream, d);
      }
    }
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  if (p.max_parts == 1) return hipSuccess;
  return launch_attn_join(d, a.dtype, a.c.tokens * a.q_heads, p.rows, stream);
}

template <typename T, bool MX>
hipError_t by_head_dim(const PagedAttentionArgs& a, hipStream_t stream) {
  if (a.c.head_dim <= 64) return run<T, MX, 64>(a, stream);
  if (a.c.head_dim <= 128) return run<T, MX, 128>(a, stream);
  return run<T, MX, 256>(a, stream);
}

}  // namespace

int64_t paged_attention_workspace(const PagedAttentionArgs& a) {
  if (a.block_count > 0) return paged_blocks_workspace(a);
  const Plan p = plan(a);
  return p.max_parts == 1 ? 0 : workspace_bytes(a, p.slots, p.rows);
}

hipError_t launch_paged_attention(const PagedAttentionArgs& a, hipStream_t stream) {
  if (a.block_count > 0) return launch_paged_blocks(a, stream);
  switch (a.dtype) {
    case kF32: return a.c.mx ? by_head_dim<float, true>(a, stream) : by_head_dim<float, false>(a, stream);
    case kF16: return a.c.mx ? by_head_dim<_Float16, true>(a, stream) : by_head_dim<_Float16, false>(a, stream);
    case kBF16: return a.c.mx ? by_head_dim<__bf16, true>(a, stream) : by_head_dim<__bf16, false>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace ako

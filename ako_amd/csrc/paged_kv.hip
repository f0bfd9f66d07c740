// Writing and reading a paged key/value cache on gfx950.
//
// paged_write: RoPE of a step's q and k at the positions that the device-side
// lengths give, q to its output, k and v into their sequences' pages, in the
// model's type or as e4m3 with a power-of-two scale per 32 elements (paged.h).
// paged_read: the same rows of both caches as dense tensors.
//
// Both move every byte once. A workgroup stays inside one token, so that the
// token's sequence, position and page are found once per wavefront and not per
// lane. Bound by HBM on long prompts: 4 x 2048 tokens into e4m3 pages, 186 MB, in
// 37.5 us, 5.0 TB/s (a copy of that size reaches 6.5); 69 MB of such pages and
// what comes of them in 15.0, 4.6 TB/s, calls one after the other. One step's 1.6 MB is
// launch latency: 2.8 us replayed from a graph.

#include <algorithm>

#include "paged.h"

namespace ako {

// Element offset of a row of the key or value pages, and of its scale codes.
// The strides are chosen by value, so that they come from scalar argument
// loads and a select, and not from vector loads of the chosen descriptor.
__device__ __forceinline__ int64_t cache_row(const PagedDev& c, bool is_v, int page, int h, int slot) {
  return page * (is_v ? c.vst[0] : c.kst[0]) + h * (is_v ? c.vst[1] : c.kst[1]) + slot * (is_v ? c.vst[2] : c.kst[2]);
}
__device__ __forceinline__ int64_t scale_row(const PagedDev& c, bool is_v, int page, int h, int slot) {
  return page * (is_v ? c.vsst[0] : c.ksst[0]) + h * (is_v ? c.vsst[1] : c.ksst[1]) +
         slot * (is_v ? c.vsst[2] : c.ksst[2]);
}

struct WriteDev {
  PagedDev c;
  const void* q;
  const void* k;
  const void* v;
  void* q_out;
  const void* cos;
  const void* sin;
  int64_t qs[3], kns[3], vns[3];  // batch, token, head strides of the new rows
  int64_t st;                     // table row stride
  int table_rows, q_heads, kv_heads, head_dim;
  int lanes;                      // lanes of a token: heads of q, k and v times per_head
  FastDiv by_blocks, by_head;     // workgroups per token, lanes per head
  int blocks, per_head, token0;
};

// Eight values of a row of the key or value pages; for e4m3 also their block's
// scale code, the block's four packets being those of a quad of lanes.
template <typename T, bool MX>
__device__ __forceinline__ void put(const PagedDev& c, bool is_v, int page, int h, int slot, int e0, const float (&r)[8], bool live) {
  const bool store = live && page >= 0;
  const int64_t base = cache_row(c, is_v, page, h, slot) + e0;
  if constexpr (MX) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = __builtin_fmaxf(m, live ? finite_abs(r[i]) : 0.0f);
    m = __builtin_fmaxf(m, dpp_mov<0xB1>(m));
    m = __builtin_fmaxf(m, dpp_mov<0x4E>(m));
    const unsigned code = e8m0_code(m);
    if (store) {
      store_bytes8(const_cast<uint8_t*>(static_cast<const uint8_t*>(is_v ? c.v : c.k)) + base, to_e4m3(r, e8m0_inverse(code)));
      if (e0 % 32 == 0)
        const_cast<uint8_t*>(is_v ? c.vs : c.ks)[scale_row(c, is_v, page, h, slot) + e0 / 32] = static_cast<uint8_t>(code);
    }
  } else if (store) {
    Eight<T> o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = from_f32<T>(r[i]);
    store_eight<T>(const_cast<T*>(static_cast<const T*>(is_v ? c.v : c.k)) + base, o);
  }
}

// q, k and v of a token are numbered through as heads, and a head's lanes
// rounded up to a multiple of four for e4m3 pages, so that a 32-element block is
// a quad of lanes and its maximum two DPP steps.
//
// What bounds the kernel at many tokens is the path from the CU's cache: a lane needs
// 64 bytes of the tables for each packet of 16. kPair lanes (neox) hold packet j
// of both halves of a head, which share those 64 bytes and are each other's
// partners; it takes halves of whole blocks for e4m3 pages (head sizes of
// 64, 128, ...): 8192 tokens of 32 + 8 heads of 128 in bfloat16 to e4m3 pages took
// 1.25 times as long with kOwn lanes. kOwn lanes hold one packet and read its partner too: the other
// sizes, and interleaved pairs, whose packets are complete in themselves.
enum WriteLayout { kOwnNeox, kPairNeox, kInterleaved };

template <typename T, typename TT, bool MX, WriteLayout LAYOUT>
__global__ __launch_bounds__(256) void paged_write(WriteDev a) {
  constexpr bool PAIR = LAYOUT == kPairNeox;
  const int nth = fast_div(blockIdx.x, a.by_blocks), token = a.token0 + nth;
  const int lane = (blockIdx.x - nth * a.blocks) * blockDim.x + threadIdx.x;
  const int head = fast_div(lane, a.by_head);
  const int e0 = (lane - head * a.per_head) * 8;
  const int half = a.head_dim / 2;
  const bool live = lane < a.lanes && e0 < (PAIR ? half : a.head_dim);
  const bool is_q = head < a.q_heads, is_v = head >= a.q_heads + a.kv_heads;
  const int h = is_q ? head : is_v ? head - a.q_heads - a.kv_heads : head - a.q_heads;

  // The rows themselves are asked for before the position is known.
  const int b = a.c.cu ? 0 : static_cast<int>(fast_div(token, a.c.by_seq));
  const int s = token - b * a.c.seq;
  const T* x = static_cast<const T*>(is_q ? a.q : is_v ? a.v : a.k);
  x += (is_q ? a.qs[0] : is_v ? a.vns[0] : a.kns[0]) * b + (is_q ? a.qs[1] : is_v ? a.vns[1] : a.kns[1]) * s +
       (is_q ? a.qs[2] : is_v ? a.vns[2] : a.kns[2]) * h;
  const bool upper = LAYOUT == kOwnNeox && e0 >= half;
  Eight<T> own = zero_eight<T>(), other = own;
  if (live) {
    own = load_eight<T, PAIR>(x + e0);
    if (PAIR) other = load_eight<T, true>(x + half + e0);
    if (LAYOUT == kOwnNeox && !is_v) other = load_eight<T>(x + (upper ? e0 - half : e0 + half));
  }

  const TokenPlace at = token_place(a.c, token);
  int slot = 0, page = -1;
  const bool known = at.seq >= 0 && at.pos >= 0 && at.pos < a.c.capacity && at.pos < a.table_rows;
  if (known) page = page_of(a.c, at.seq, at.pos, slot);

  float r[8], r2[8];
  if (live && !is_v && page >= 0) {
    if constexpr (LAYOUT != kInterleaved) {
      float c[8], n[8];
      const int64_t row = at.pos * a.st + (upper ? e0 - half : e0);
      load_f32<TT, 8>(static_cast<const TT*>(a.cos) + row, c);
      load_f32<TT, 8>(static_cast<const TT*>(a.sin) + row, n);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float o = to_f32(own[i]), p = to_f32(other[i]);
        r[i] = upper ? p * n[i] + o * c[i] : o * c[i] - p * n[i];
        r2[i] = o * n[i] + p * c[i];
      }
    } else {
      float c[4], n[4];
      const int64_t row = at.pos * a.st + e0 / 2;
      load_f32<TT, 4>(static_cast<const TT*>(a.cos) + row, c);
      load_f32<TT, 4>(static_cast<const TT*>(a.sin) + row, n);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float o = to_f32(own[2 * i]), p = to_f32(own[2 * i + 1]);
        r[2 * i] = o * c[i] - p * n[i];
        r[2 * i + 1] = o * n[i] + p * c[i];
      }
    }
  } else {
    // A row without a slot: q is zero where there is no such token, and NaN
    // where the token lies outside the cache or the tables.
    const float fill = at.seq < 0 || at.pos < 0 ? 0.0f : __builtin_nanf("");
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      r[i] = is_v ? to_f32(own[i]) : fill;
      r2[i] = is_v ? to_f32(other[i]) : fill;
    }
  }

  if (is_q && live) {
    T* const out = static_cast<T*>(a.q_out) + (int64_t(token) * a.q_heads + h) * a.head_dim + e0;
    Eight<T> o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = from_f32<T>(r[i]);
    store_eight<T, true>(out, o);
    if constexpr (PAIR) {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = from_f32<T>(r2[i]);
      store_eight<T, true>(out + half, o);
    }
  }
  if (!MX && is_q) return;  // e4m3: every lane takes part in its quad's maximum
  put<T, MX>(a.c, is_v, page, h, slot, e0, r, live && !is_q);
  if constexpr (PAIR) put<T, MX>(a.c, is_v, page, h, slot, e0 + half, r2, live && !is_q);
}

struct ReadDev {
  PagedDev c;
  void* k_out;
  void* v_out;
  int kv_heads, head_dim;
  int lanes;                   // lanes of a token: heads of k and v times head_dim / 8
  FastDiv by_blocks, by_head;
  int blocks, per_head, token0;
};

// A lane moves eight elements: its store is 16 bytes of a half type, and a
// wavefront's stores are one run. Sixteen elements of e4m3 a lane, in one load
// and two stores 32 bytes apart, took 1.3 times as long, and stores without the
// non-temporal hint 1.1 times (16 sequences of up to 4096 positions, 8 heads of 128, e4m3
// to bfloat16, 69 MB).
template <typename T, bool MX>
__global__ __launch_bounds__(256) void paged_read(ReadDev a) {
  const int nth = fast_div(blockIdx.x, a.by_blocks), token = a.token0 + nth;
  const int lane = (blockIdx.x - nth * a.blocks) * blockDim.x + threadIdx.x;
  const int head = fast_div(lane, a.by_head);
  const int e0 = (lane - head * a.per_head) * 8;
  const bool is_v = head >= a.kv_heads;
  const int h = is_v ? head - a.kv_heads : head;
  const TokenPlace at = token_place(a.c, token);
  int slot = 0, page = -1;
  if (at.seq >= 0 && at.pos >= 0 && at.pos < a.c.capacity) page = page_of(a.c, at.seq, at.pos, slot);
  if (lane >= a.lanes) return;
  Eight<T> o = zero_eight<T>();
  if (page >= 0) {
    const int64_t base = cache_row(a.c, is_v, page, h, slot) + e0;
    if constexpr (MX) {
      const unsigned code = (is_v ? a.c.vs : a.c.ks)[scale_row(a.c, is_v, page, h, slot) + e0 / 32];
      o = from_e4m3<T>(load_bytes8(static_cast<const uint8_t*>(is_v ? a.c.v : a.c.k) + base), e8m0_scale(code));
    } else {
      o = load_eight<T, true>(static_cast<const T*>(is_v ? a.c.v : a.c.k) + base);
    }
  }
  store_eight<T, true>(static_cast<T*>(is_v ? a.v_out : a.k_out) + (int64_t(token) * a.kv_heads + h) * a.head_dim + e0, o);
}

namespace {

// Workgroups of a token: the size of 64 to 256 lanes that leaves the fewest idle.
int block_size(int lanes) {
  int best = 256;
  for (int b = 256; b >= 64; b -= 64)
    if (ceil_div(lanes, b) * b < ceil_div(lanes, best) * best) best = b;
  return best;
}

// Launches of at most 2^22 workgroups (work-items stay below 2^32), whole tokens each.
template <typename Launch>
hipError_t by_tokens(int64_t tokens, int64_t blocks, Launch launch) {
  const int64_t per = std::max<int64_t>(1, (int64_t(1) << 22) / blocks);
  for (int64_t t = 0; t < tokens; t += per) {
    launch(static_cast<int>(t), dim3(static_cast<unsigned>(std::min(per, tokens - t) * blocks)));
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  return hipSuccess;
}

template <typename T, typename TT, bool MX>
hipError_t run_write(const PagedWriteArgs& a, hipStream_t stream) {
  WriteDev d{};
  d.c = paged_dev(a.c);
  d.q = a.q;
  d.k = a.k;
  d.v = a.v;
  d.q_out = a.q_out;
  d.cos = a.cos;
  d.sin = a.sin;
  for (int i = 0; i < 3; ++i) {
    d.qs[i] = a.qs[i];
    d.kns[i] = a.kns[i];
    d.vns[i] = a.vns[i];
  }
  d.st = a.st;
  d.table_rows = static_cast<int>(std::min<int64_t>(a.table_rows, a.c.table_width * a.c.page_size));
  d.q_heads = static_cast<int>(a.q_heads);
  d.kv_heads = static_cast<int>(a.c.kv_heads);
  d.head_dim = static_cast<int>(a.c.head_dim);
  const bool pair = a.neox && (!MX || d.head_dim % 64 == 0);
  d.per_head = d.head_dim / (pair ? 16 : 8);
  if (MX) d.per_head = static_cast<int>(ceil_div(d.per_head, 4) * 4);
  d.lanes = (d.q_heads + 2 * d.kv_heads) * d.per_head;
  const int block = block_size(d.lanes);
  d.blocks = static_cast<int>(ceil_div(d.lanes, block));
  d.by_blocks = make_fastdiv(d.blocks);
  d.by_head = make_fastdiv(d.per_head);
  return by_tokens(a.c.tokens, d.blocks, [&](int token0, dim3 grid) {
    d.token0 = token0;
    if (pair) AKO_LAUNCH((paged_write<T, TT, MX, kPairNeox>), grid, dim3(block), 0, stream, d);
    else if (!a.neox) AKO_LAUNCH((paged_write<T, TT, MX, kInterleaved>), grid, dim3(block), 0, stream, d);
    else if constexpr (MX) AKO_LAUNCH((paged_write<T, TT, MX, kOwnNeox>), grid, dim3(block), 0, stream, d);
  });
}

template <typename T, bool MX>
hipError_t write_tables(const PagedWriteArgs& a, hipStream_t stream) {
  switch (a.table_dtype) {
    case kF32: return run_write<T, float, MX>(a, stream);
    case kF16: return run_write<T, _Float16, MX>(a, stream);
    case kBF16: return run_write<T, __bf16, MX>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

template <typename T>
hipError_t run_read(const PagedReadArgs& a, hipStream_t stream) {
  ReadDev d{};
  d.c = paged_dev(a.c);
  d.k_out = a.k_out;
  d.v_out = a.v_out;
  d.kv_heads = static_cast<int>(a.c.kv_heads);
  d.head_dim = static_cast<int>(a.c.head_dim);
  d.per_head = d.head_dim / 8;
  d.lanes = 2 * d.kv_heads * d.per_head;
  const int block = block_size(d.lanes);
  d.blocks = static_cast<int>(ceil_div(d.lanes, block));
  d.by_blocks = make_fastdiv(d.blocks);
  d.by_head = make_fastdiv(d.per_head);
  return by_tokens(a.c.tokens, d.blocks, [&](int token0, dim3 grid) {
    d.token0 = token0;
    if (a.c.mx) AKO_LAUNCH((paged_read<T, true>), grid, dim3(block), 0, stream, d);
    else AKO_LAUNCH((paged_read<T, false>), grid, dim3(block), 0, stream, d);
  });
}

}  // namespace

hipError_t launch_paged_write(const PagedWriteArgs& a, hipStream_t stream) {
  const bool mx = a.c.mx;
  switch (a.dtype) {
    case kF32: return mx ? write_tables<float, true>(a, stream) : write_tables<float, false>(a, stream);
    case kF16: return mx ? write_tables<_Float16, true>(a, stream) : write_tables<_Float16, false>(a, stream);
    case kBF16: return mx ? write_tables<__bf16, true>(a, stream) : write_tables<__bf16, false>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_paged_read(const PagedReadArgs& a, hipStream_t stream) {
  switch (a.dtype) {
    case kF32: return run_read<float>(a, stream);
    case kF16: return run_read<_Float16>(a, stream);
    case kBF16: return run_read<__bf16>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace ako

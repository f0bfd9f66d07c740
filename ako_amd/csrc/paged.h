// What the kernels over a paged key/value cache share: where a sequence's
// positions lie, which sequence a token row belongs to, and the 8-bit format.
//
// Nothing that comes from device memory is trusted with an address: a length
// is clamped to the positions the block table can name, a page outside the
// pool counts as absent, and a token row outside its sequence as padding.
#pragma once

#include "common.h"
#include "launch.h"

namespace ako {

// ---- which sequence a token row belongs to ----------------------------------
struct PagedDev {
  const void* k;
  const void* v;
  const uint8_t* ks;  // E8M0 scale codes of e4m3 pages, else null
  const uint8_t* vs;
  const int* table;
  const int* lens;
  const int* cu;        // null: every sequence has `seq` tokens
  int64_t kst[3], vst[3];    // page, head, slot strides in elements
  int64_t ksst[3], vsst[3];  // the same of the scale codes
  int64_t table_stride;
  int n_seqs, num_pages, page_size, capacity;  // capacity: positions a table row can name
  int tokens, seq;
  FastDiv by_seq, by_page;
};

inline PagedDev paged_dev(const PagedArgs& a) {
  PagedDev d{};
  d.k = a.k;
  d.v = a.v;
  d.ks = static_cast<const uint8_t*>(a.ks);
  d.vs = static_cast<const uint8_t*>(a.vs);
  d.table = a.table;
  d.lens = a.lens;
  d.cu = a.cu;
  for (int i = 0; i < 3; ++i) {
    d.kst[i] = a.kst[i];
    d.vst[i] = a.vst[i];
    d.ksst[i] = a.ksst[i];
    d.vsst[i] = a.vsst[i];
  }
  d.table_stride = a.table_stride;
  d.n_seqs = static_cast<int>(a.n_seqs);
  d.num_pages = static_cast<int>(a.num_pages);
  d.page_size = static_cast<int>(a.page_size);
  d.capacity = a.num_pages > 0 ? static_cast<int>(a.table_width * a.page_size) : 0;
  d.tokens = static_cast<int>(a.tokens);
  d.seq = a.cu || a.n_seqs == 0 ? 0 : static_cast<int>(a.tokens / a.n_seqs);
  d.by_seq = make_fastdiv(d.seq > 0 ? d.seq : 1);
  d.by_page = make_fastdiv(d.page_size);
  return d;
}

// The largest i in [0, n] with key(i) <= x, for key(0) <= x and key ascending:
// 64 keys are compared at a time, one per lane. x is the same in every lane,
// and all 64 lanes take part.
template <typename Key>
__device__ __forceinline__ int last_at_most(int n, int x, Key key) {
  const int lane = threadIdx.x % kWave;
  int found = 0;
  for (int base = 0; base <= n; base += kWave) {
    const int i = base + lane;
    found += __popcll(__ballot(i <= n && key(i) <= x));
  }
  return found > 0 ? found - 1 : 0;
}

// One token row's place: sequence (-1: a row behind the last sequence) and
// position, negative where the sequence has fewer positions than new tokens.
struct TokenPlace {
  int seq, pos;
};

__device__ __forceinline__ TokenPlace token_place(const PagedDev& p, int token) {
  if (p.cu == nullptr) {
    if (p.seq == 0) return TokenPlace{-1, -1};
    const int s = fast_div(token, p.by_seq);
    return TokenPlace{s, max(p.lens[s], 0) - p.seq + (token - s * p.seq)};
  }
  const int s = last_at_most(p.n_seqs, token, [&](int i) { return p.cu[i]; });
  if (s >= p.n_seqs) return TokenPlace{-1, -1};
  const int first = p.cu[s], end = p.cu[s + 1];
  if (token < first || token >= end) return TokenPlace{-1, -1};
  return TokenPlace{s, max(p.lens[s], 0) - (end - token)};
}

// The page that holds position pos of sequence s, or -1.
__device__ __forceinline__ int page_of(const PagedDev& p, int s, int pos, int& slot) {
  const int at = fast_div(pos, p.by_page);
  slot = pos - at * p.page_size;
  const int page = p.table[s * p.table_stride + at];
  return page >= 0 && page < p.num_pages ? page : -1;
}

// ---- e4m3 rows with a power-of-two scale per 32 elements -----------------------
// An E8M0 code c stands for 2^(c - 127), 255 for NaN. A block's code is the smallest under
// which no finite element passes e4m3's largest value, 448 = 1.75 * 2^8; so
// nothing is clipped, and every element at or above 2^-6 of its scale is off
// by at most half a step of e4m3, 2^-4 of itself. Codes below 1 are not used:
// scales and their reciprocals stay normal floats. Infinities and NaN become
// e4m3's NaN and do not count for the scale.
__device__ __forceinline__ unsigned e8m0_code(float amax) {
  const unsigned bits = __builtin_bit_cast(unsigned, amax);
  const int e = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u);
  return static_cast<unsigned>(max(e, -126) + 127);
}
constexpr unsigned kUnitCode = 127;
__device__ __forceinline__ float e8m0_scale(unsigned code) { return __builtin_bit_cast(float, code << 23); }
__device__ __forceinline__ float e8m0_inverse(unsigned code) { return __builtin_bit_cast(float, (254u - code) << 23); }

__device__ __forceinline__ float finite_abs(float v) {
  const float m = __builtin_fabsf(v);
  return m < __builtin_inff() ? m : 0.0f;  // NaN compares false
}

// Eight floats times `inv` as e4m3, round to nearest even.
__device__ __forceinline__ u32x2 to_e4m3(const float (&x)[8], float inv) {
  u32x2 q;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * w] * inv, x[4 * w + 1] * inv, 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * w + 2] * inv, x[4 * w + 3] * inv, r, true);
    q[w] = static_cast<unsigned>(r);
  }
  return q;
}

// Four e4m3 values (one word) times a power of two as T. Exact for float and
// __bf16; for _Float16 where the value is in its range (beyond it infinite,
// below its normal range rounded).
template <typename T> struct FromE4m3;
template <> struct FromE4m3<float> {
  typedef float v2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ v2 lo(unsigned w, float s) { return __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, s, false); }
  static __device__ __forceinline__ v2 hi(unsigned w, float s) { return __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, s, true); }
};
template <> struct FromE4m3<_Float16> {
  typedef _Float16 v2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ v2 lo(unsigned w, float s) { return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, false); }
  static __device__ __forceinline__ v2 hi(unsigned w, float s) { return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, true); }
};
template <> struct FromE4m3<__bf16> {
  typedef __bf16 v2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ v2 lo(unsigned w, float s) { return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, false); }
  static __device__ __forceinline__ v2 hi(unsigned w, float s) { return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, true); }
};

// Eight elements of T.
template <typename T>
struct Eight {
  static constexpr int kPer = 16 / static_cast<int>(sizeof(T));
  Pack<T, kPer> p[8 / kPer];
  __device__ __forceinline__ T& operator[](int i) { return p[i / kPer].e[i % kPer]; }
  __device__ __forceinline__ const T& operator[](int i) const { return p[i / kPer].e[i % kPer]; }
};

template <typename T, bool NT = false>
__device__ __forceinline__ Eight<T> load_eight(const T* p) {
  Eight<T> r;
#pragma unroll
  for (int c = 0; c < 8 / Eight<T>::kPer; ++c) r.p[c] = load_pack<T, Eight<T>::kPer, NT>(p + c * Eight<T>::kPer);
  return r;
}
template <typename T, bool NT = false>
__device__ __forceinline__ void store_eight(T* p, const Eight<T>& r) {
#pragma unroll
  for (int c = 0; c < 8 / Eight<T>::kPer; ++c) store_pack<T, Eight<T>::kPer, NT>(p + c * Eight<T>::kPer, r.p[c]);
}
template <typename T>
__device__ __forceinline__ Eight<T> zero_eight() {
  Eight<T> r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = from_f32<T>(0.0f);
  return r;
}

template <typename T>
__device__ __forceinline__ Eight<T> from_e4m3(u32x2 q, float scale) {
  Eight<T> r;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const auto a = FromE4m3<T>::lo(q[w], scale), b = FromE4m3<T>::hi(q[w], scale);
    r[4 * w] = a[0];
    r[4 * w + 1] = a[1];
    r[4 * w + 2] = b[0];
    r[4 * w + 3] = b[1];
  }
  return r;
}

// Eight bytes at any alignment.
__device__ __forceinline__ u32x2 load_bytes8(const uint8_t* p) {
  typedef u32x2 mem_t __attribute__((aligned(1)));
  return *reinterpret_cast<const mem_t*>(p);
}
__device__ __forceinline__ void store_bytes8(uint8_t* p, u32x2 v) {
  typedef u32x2 mem_t __attribute__((aligned(1)));
  *reinterpret_cast<mem_t*>(p) = v;
}

}  // namespace ako

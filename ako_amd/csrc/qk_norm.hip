// RMSNorm of every head of q and k, and RoPE, in one pass on gfx950.
//
//   y = (x * rsqrt(sum(x^2) / head_dim + eps)) * w      for each head, w per element
//   (a, b) -> (a c - b n, a n + b c)                    for each rotated pair of y
//
// in 32 bits, a rotated element in two roundings, the result rounded once to the
// storage type: nothing is rounded between the norm and the rotation, as it is
// where two operators follow each other.
//
// A head is a group of L lanes, L a power of two, so that its sum of squares is
// log2(L) steps inside the wavefront and nothing is staged anywhere. A lane
// holds two packets of 16 bytes, neox those that are each other's partners
// (packet j of both halves), interleaved 32 bytes in a row. Where a half is no
// whole number of packets the last one is moved back to end with it; what that
// repeats is left out of the sum and stored twice with the same values.
//
// Bound by HBM: 4 x 2048 tokens of 32 + 8 heads of 128 in bfloat16, 169 MB, in 28.2 us, 6.0 TB/s.

#include <algorithm>

#include "common.h"
#include "launch.h"

namespace ako {

struct NormRopeDev {
  const void* q;
  const void* k;
  const void* qw;
  const void* kw;
  const void* cos;
  const void* sin;
  void* q_out;
  void* k_out;
  int64_t qs[3], ks[3];  // batch, token, head strides
  int64_t st;            // table row stride
  int64_t token0;
  unsigned units;        // heads of all tokens in this launch
  int q_heads, k_heads, head_dim;
  int lanes_log2;        // of a head
  float eps, inv_dim;
  FastDiv by_heads, by_seq;
  int seq;
};

template <typename T, typename TT, typename WT, bool NEOX, int E>
__global__ __launch_bounds__(256) void norm_rope(NormRopeDev a) {
  const unsigned id = blockIdx.x * blockDim.x + threadIdx.x;
  unsigned unit = id >> a.lanes_log2;
  const int j = id & ((1 << a.lanes_log2) - 1), half = a.head_dim / 2;
  const bool live = unit < a.units && j * E < half;
  unit = min(unit, a.units - 1);
  const unsigned nth = fast_div(unit, a.by_heads);
  const int head = unit - nth * (a.q_heads + a.k_heads);
  const unsigned token = static_cast<unsigned>(a.token0) + nth;
  const unsigned b = fast_div(token, a.by_seq), s = token - b * a.seq;
  const bool is_q = head < a.q_heads;
  const int h = is_q ? head : head - a.q_heads;

  // The packets' first elements in the head, and the table's. `fresh`: the first element
  // of them that the lane before does not hold.
  const int step = NEOX ? E : 2 * E, whole = NEOX ? half : a.head_dim;
  const int at = max(0, min(j * step, whole - step)), fresh = j * step - at;
  const int second = NEOX ? at + half : at + E, row = NEOX ? at : at / 2;
  const T* x = static_cast<const T*>(is_q ? a.q : a.k) + (is_q ? a.qs[0] : a.ks[0]) * b + (is_q ? a.qs[1] : a.ks[1]) * s +
               (is_q ? a.qs[2] : a.ks[2]) * h;
  const Pack<T, E> p0 = load_pack<T, E, true>(x + at), p1 = load_pack<T, E, true>(x + second);
  float c[E], n[E], w0[E], w1[E];
  load_f32<TT, E>(static_cast<const TT*>(a.cos) + s * a.st + row, c);
  load_f32<TT, E>(static_cast<const TT*>(a.sin) + s * a.st + row, n);
  const WT* w = static_cast<const WT*>(is_q ? a.qw : a.kw);
  load_f32<WT, E>(w + at, w0);
  load_f32<WT, E>(w + second, w1);

  float x0[E], x1[E], ss = 0.0f;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    x0[i] = to_f32(p0.e[i]);
    x1[i] = to_f32(p1.e[i]);
    if (live && i >= fresh) ss = __builtin_fmaf(x0[i], x0[i], ss);
    if (live && (NEOX ? i : E + i) >= fresh) ss = __builtin_fmaf(x1[i], x1[i], ss);
  }
  const float r = inverse_rms(lane_group_sum(ss, a.lanes_log2), a.inv_dim, a.eps);
#pragma unroll
  for (int i = 0; i < E; ++i) {
    x0[i] = x0[i] * r * w0[i];
    x1[i] = x1[i] * r * w1[i];
  }
  Pack<T, E> y0, y1;
  if constexpr (NEOX || E == 1) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      y0.e[i] = from_f32<T>(__builtin_fmaf(x0[i], c[i], -(x1[i] * n[i])));
      y1.e[i] = from_f32<T>(__builtin_fmaf(x0[i], n[i], x1[i] * c[i]));
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      y0.e[i] = from_f32<T>(__builtin_fmaf(x0[i], c[i / 2], -(x0[i + 1] * n[i / 2])));
      y0.e[i + 1] = from_f32<T>(__builtin_fmaf(x0[i], n[i / 2], x0[i + 1] * c[i / 2]));
      y1.e[i] = from_f32<T>(__builtin_fmaf(x1[i], c[E / 2 + i / 2], -(x1[i + 1] * n[E / 2 + i / 2])));
      y1.e[i + 1] = from_f32<T>(__builtin_fmaf(x1[i], n[E / 2 + i / 2], x1[i + 1] * c[E / 2 + i / 2]));
    }
  }
  if (!live) return;
  T* y = is_q ? static_cast<T*>(a.q_out) + (int64_t(token) * a.q_heads + h) * a.head_dim
              : static_cast<T*>(a.k_out) + (int64_t(token) * a.k_heads + h) * a.head_dim;
  store_pack<T, E, true>(y + at, y0);
  store_pack<T, E, true>(y + second, y1);
}

namespace {

template <typename T, typename TT, typename WT, bool NEOX, int E>
hipError_t run_packets(const NormRopeArgs& a, hipStream_t stream) {
  NormRopeDev d{};
  d.q = a.q;
  d.k = a.k;
  d.qw = a.qw;
  d.kw = a.kw;
  d.cos = a.cos;
  d.sin = a.sin;
  d.q_out = a.q_out;
  d.k_out = a.k_out;
  for (int i = 0; i < 3; ++i) {
    d.qs[i] = a.qs[i];
    d.ks[i] = a.ks[i];
  }
  d.st = a.st;
  d.q_heads = static_cast<int>(a.q_heads);
  d.k_heads = static_cast<int>(a.k_heads);
  d.head_dim = static_cast<int>(a.head_dim);
  while ((int64_t(E) << d.lanes_log2) < a.head_dim / 2) ++d.lanes_log2;
  d.eps = a.eps;
  d.inv_dim = 1.0f / static_cast<float>(a.head_dim);
  d.seq = static_cast<int>(a.seq);
  d.by_heads = make_fastdiv(d.q_heads + d.k_heads);
  d.by_seq = make_fastdiv(d.seq);
  // A launch's lanes stay below 2^30, whole tokens each.
  const int64_t heads = a.q_heads + a.k_heads, tokens = a.batch * a.seq;
  const int64_t per = std::max<int64_t>(1, (int64_t(1) << 30) / (heads << d.lanes_log2));
  for (int64_t t = 0; t < tokens; t += per) {
    const int64_t units = std::min(per, tokens - t) * heads;
    d.token0 = t;
    d.units = static_cast<unsigned>(units);
    AKO_LAUNCH((norm_rope<T, TT, WT, NEOX, E>), dim3(static_cast<unsigned>(ceil_div(units << d.lanes_log2, 256))), dim3(256), 0,
               stream, d);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  return hipSuccess;
}

template <typename T, typename TT, typename WT>
hipError_t run_weights(const NormRopeArgs& a, hipStream_t stream) {
  constexpr int E = 16 / sizeof(T);
  const bool packets = a.head_dim / 2 >= E;
  if (a.neox) return packets ? run_packets<T, TT, WT, true, E>(a, stream) : run_packets<T, TT, WT, true, 1>(a, stream);
  return packets ? run_packets<T, TT, WT, false, E>(a, stream) : run_packets<T, TT, WT, false, 1>(a, stream);
}

template <typename T, typename TT>
hipError_t run_tables(const NormRopeArgs& a, hipStream_t stream) {
  if (a.w_dtype == a.dtype) return run_weights<T, TT, T>(a, stream);
  return run_weights<T, TT, float>(a, stream);
}

template <typename T>
hipError_t run_rows(const NormRopeArgs& a, hipStream_t stream) {
  switch (a.table_dtype) {
    case kF32: return run_tables<T, float>(a, stream);
    case kF16: return run_tables<T, _Float16>(a, stream);
    case kBF16: return run_tables<T, __bf16>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

hipError_t launch_norm_rope(const NormRopeArgs& a, hipStream_t stream) {
  switch (a.dtype) {
    case kF32: return run_rows<float>(a, stream);
    case kF16: return run_rows<_Float16>(a, stream);
    case kBF16: return run_rows<__bf16>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace ako

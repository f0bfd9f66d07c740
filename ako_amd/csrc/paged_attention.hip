// Attention of a step's tokens over a paged key/value cache on gfx950.
//
// Token row t at position p of its sequence sees the keys j <= p, and with a
// window w only those with j > p - w or j < sinks:
//   out = sum_j e^(scale q.k_j - m) v_j / sum_j e^(scale q.k_j - m),  m = max_j scale q.k_j
// in 32 bits, zero where nothing is visible.

#include <algorithm>
#include <limits>

#include "paged.h"

namespace ako {

struct AttnDev {
  PagedDev c;
  const void* q;
  void* out;
  int64_t qs[3];
  int q_heads, group, head_dim;
  int window, sinks;
  float scale_log2;  // scale * log2(e)
  FastDiv by_heads, by_group;
};

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int m = 1; m < kWave; m *= 2) v = __builtin_fmaxf(v, __shfl_xor(v, m));
  return v;
}

// One wavefront per (token, query head): 64 keys at a time, one key per lane
// for the products, then one slice of the head per lane for the sum.
template <typename T, bool MX>
__global__ __launch_bounds__(kWave) void paged_attention_simple(AttnDev a) {
  __shared__ float qv[256], pv[kWave];
  __shared__ int64_t row[kWave];
  __shared__ int64_t srow[kWave];
  const int lane = threadIdx.x;
  const int token = fast_div(blockIdx.x, a.by_heads), h = blockIdx.x - token * a.q_heads;
  const int kvh = fast_div(h, a.by_group);
  const TokenPlace at = token_place(a.c, token);
  const int b = a.c.cu ? 0 : static_cast<int>(fast_div(token, a.c.by_seq));
  const T* q = static_cast<const T*>(a.q) + b * a.qs[0] + (token - b * a.c.seq) * a.qs[1] + h * a.qs[2];
  for (int d = lane; d < a.head_dim; d += kWave) qv[d] = to_f32(q[d]);
  __syncthreads();
  float m = -__builtin_inff(), l = 0.0f, acc[4] = {};
  const int end = at.seq < 0 ? 0 : min(at.pos + 1, a.c.capacity);
  const int low = a.window > 0 ? max(0, at.pos - a.window + 1) : 0;
  for (int j0 = 0; j0 < end; j0 += kWave) {
    if (j0 + kWave <= low && j0 >= a.sinks) continue;
    const int j = j0 + lane;
    int slot = 0, page = -1;
    const bool seen = j < end && (j >= low || j < a.sinks);
    if (seen) page = page_of(a.c, at.seq, j, slot);
    float s = -__builtin_inff();
    if (page >= 0) {
      s = 0.0f;
      const int64_t kr = page * a.c.kst[0] + kvh * a.c.kst[1] + slot * a.c.kst[2];
      const int64_t sr = MX ? page * a.c.ksst[0] + kvh * a.c.ksst[1] + slot * a.c.ksst[2] : 0;
      for (int d = 0; d < a.head_dim; d += 8) {
        Eight<T> x;
        if constexpr (MX) x = from_e4m3<T>(load_bytes8(static_cast<const uint8_t*>(a.c.k) + kr + d), e8m0_scale(a.c.ks[sr + d / 32]));
        else x = load_eight<T>(static_cast<const T*>(a.c.k) + kr + d);
#pragma unroll
        for (int i = 0; i < 8; ++i) s = __builtin_fmaf(qv[d + i], to_f32(x[i]), s);
      }
      s *= a.scale_log2;
    }
    row[lane] = page < 0 ? -1 : page * a.c.vst[0] + kvh * a.c.vst[1] + slot * a.c.vst[2];
    srow[lane] = page < 0 || !MX ? 0 : page * a.c.vsst[0] + kvh * a.c.vsst[1] + slot * a.c.vsst[2];
    const float top = wave_max(s), mn = __builtin_fmaxf(m, top);
    const float base = mn == -__builtin_inff() ? 0.0f : mn;
    const float p = page < 0 ? 0.0f : __builtin_amdgcn_exp2f(s - base), keep = __builtin_amdgcn_exp2f(m - base);
    pv[lane] = p;
    l = l * keep + wave_sum(p);
    m = mn;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] *= keep;
    for (int k = 0; k < kWave; ++k) {
      if (row[k] < 0) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = lane + kWave * i;
        if (d >= a.head_dim) continue;
        float v;
        if constexpr (MX) {
          const unsigned w = static_cast<const uint8_t*>(a.c.v)[row[k] + d];
          v = to_f32(static_cast<T>(FromE4m3<T>::lo(w, e8m0_scale(a.c.vs[srow[k] + d / 32]))[0]));
        } else {
          v = to_f32(static_cast<const T*>(a.c.v)[row[k] + d]);
        }
        acc[i] = __builtin_fmaf(pv[k], v, acc[i]);
      }
    }
    __syncthreads();
  }
  T* out = static_cast<T*>(a.out) + (int64_t(token) * a.q_heads + h) * a.head_dim;
  const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = lane + kWave * i;
    if (d < a.head_dim) out[d] = from_f32<T>(acc[i] * inv);
  }
}

namespace {

template <typename T>
hipError_t run(const PagedAttentionArgs& a, hipStream_t stream) {
  AttnDev d{};
  d.c = paged_dev(a.c);
  d.q = a.q;
  d.out = a.out;
  for (int i = 0; i < 3; ++i) d.qs[i] = a.qs[i];
  d.q_heads = static_cast<int>(a.q_heads);
  d.group = static_cast<int>(a.q_heads / a.c.kv_heads);
  d.head_dim = static_cast<int>(a.c.head_dim);
  const int64_t most = std::numeric_limits<int>::max();
  d.window = static_cast<int>(std::min(a.window, most));
  d.sinks = static_cast<int>(std::min(a.sinks, most));
  d.scale_log2 = a.scale * 1.44269504088896340736f;
  d.by_heads = make_fastdiv(d.q_heads);
  d.by_group = make_fastdiv(d.group);
  const dim3 grid(static_cast<unsigned>(a.c.tokens * a.q_heads));
  if (a.c.mx) AKO_LAUNCH((paged_attention_simple<T, true>), grid, dim3(kWave), 0, stream, d);
  else AKO_LAUNCH((paged_attention_simple<T, false>), grid, dim3(kWave), 0, stream, d);
  return hipGetLastError();
}

}  // namespace

int64_t paged_attention_workspace(const PagedAttentionArgs&) { return 0; }

hipError_t launch_paged_attention(const PagedAttentionArgs& a, hipStream_t stream) {
  switch (a.dtype) {
    case kF32: return run<float>(a, stream);
    case kF16: return run<_Float16>(a, stream);
    case kBF16: return run<__bf16>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace ako

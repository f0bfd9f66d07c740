// The C ABI (include/ako_hip.h): argument validation, status codes, and the
// hand-off to the kernel launchers. Validation runs entirely on the host and
// before any HIP call, so every rejection path is testable on a machine
// without a GPU.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <limits>
#include <string>

#include "ako_hip.h"
#include "common.h"
#include "launch.h"

namespace {

thread_local std::string g_last_error;

int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  std::vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_last_error = buf;
  return code;
}

int hip_status(hipError_t err, const char* what) {
  if (err == hipSuccess) return AKO_OK;
  if (err == hipErrorNoDevice || err == hipErrorInvalidDevice)
    return fail(AKO_ERR_NO_DEVICE, "%s: %s", what, hipGetErrorString(err));
  return fail(AKO_ERR_HIP, "%s: %s", what, hipGetErrorString(err));
}

bool valid_dtype(int dt) { return dt == AKO_DTYPE_F32 || dt == AKO_DTYPE_F16 || dt == AKO_DTYPE_BF16; }

const char* dtype_name(int dt) {
  switch (dt) {
    case AKO_DTYPE_F32: return "f32";
    case AKO_DTYPE_F16: return "f16";
    case AKO_DTYPE_BF16: return "bf16";
    default: return "?";
  }
}

bool aligned(const void* p, int64_t bytes) {
  return (reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(bytes)) == 0;
}

// Byte range [lo, hi) spanned by `count` rows of `width` elements, `stride`
// apart. `ok` is false when the extent exceeds 2^56 bytes or wraps the address
// space (sizes no allocation can have); the arithmetic is done in 128 bits so
// that such arguments cannot wrap into a small, plausible-looking span.
constexpr __int128 kMaxSpanBytes = static_cast<__int128>(1) << 56;

struct Span {
  uintptr_t lo = 0, hi = 0;
  bool ok = true;
};

Span span_bytes(const void* p, __int128 bytes) {
  Span s;
  s.lo = reinterpret_cast<uintptr_t>(p);
  if (bytes < 0 || bytes > kMaxSpanBytes) {
    s.ok = false;
    s.hi = s.lo;
    return s;
  }
  s.hi = s.lo + static_cast<uintptr_t>(bytes);
  s.ok = s.hi >= s.lo;
  return s;
}

Span span_2d(const void* p, int64_t rows, int64_t width, int64_t stride, int elem) {
  const __int128 last = static_cast<__int128>(rows - 1) * stride + width;
  return span_bytes(p, last * elem);
}

bool overlap(const Span& a, const Span& b) { return a.lo < b.hi && b.lo < a.hi; }

constexpr int64_t kMaxInt = std::numeric_limits<int32_t>::max();

}  // namespace

extern "C" {

int ako_abi_version(void) { return AKO_ABI_VERSION; }

int ako_hip_runtime_version(void) {
  int v = 0;
  if (hipRuntimeGetVersion(&v) != hipSuccess) return -1;
  return v;
}

const char* ako_build_info(void) {
  static const std::string info = std::string("ako_hip abi=") + std::to_string(AKO_ABI_VERSION) +
                                  " arch=gfx950 hip_headers=" + std::to_string(HIP_VERSION);
  return info.c_str();
}

const char* ako_last_error(void) { return g_last_error.c_str(); }

int ako_device_identity(int device, char* buf, int64_t buf_len) {
  const char* fn = "ako_device_identity";
  if (buf == nullptr || buf_len <= 0) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: no output buffer", fn);
  hipDeviceProp_t props;
  const hipError_t err = hipGetDeviceProperties(&props, device);
  if (err != hipSuccess) return hip_status(err, fn);
  int driver = 0;
  if (hipDriverGetVersion(&driver) != hipSuccess) driver = -1;
  props.name[sizeof(props.name) - 1] = '\0';
  props.gcnArchName[sizeof(props.gcnArchName) - 1] = '\0';
  const int n = std::snprintf(buf, static_cast<size_t>(buf_len),
                              "name=%s;arch=%s;cus=%d;clock_khz=%d;mem_bytes=%llu;hip_driver=%d", props.name,
                              props.gcnArchName, props.multiProcessorCount, props.clockRate,
                              static_cast<unsigned long long>(props.totalGlobalMem), driver);
  if (n < 0 || n >= buf_len) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: buffer of %lld bytes is too small", fn,
                                         static_cast<long long>(buf_len));
  return AKO_OK;
}

int ako_time_next_launch(void* start_event, void* stop_event) {
  if ((start_event == nullptr) != (stop_event == nullptr))
    return fail(AKO_ERR_INVALID_ARGUMENT, "ako_time_next_launch: start and stop must both be set or both be NULL");
  ako::ArmedEvents& slot = ako::armed_events();
  if (start_event == nullptr) {
    const bool pending = slot.start != nullptr;
    slot = ako::ArmedEvents{};
    return pending ? 1 : AKO_OK;
  }
  slot.start = static_cast<hipEvent_t>(start_event);
  slot.stop = static_cast<hipEvent_t>(stop_event);
  return AKO_OK;
}

int ako_set_tuning(int op, int key, int value) {
  if (value < 0) return fail(AKO_ERR_INVALID_ARGUMENT, "tuning value must be >= 0, got %d", value);
  switch (op) {
    case 0:
      if (key == 1) { ako::g_rms_tuning.waves_per_row = value; return AKO_OK; }
      if (key == 2) { ako::g_rms_tuning.vecs_per_thread = value; return AKO_OK; }
      if (key == 3) { ako::g_rms_tuning.force_stream = value; return AKO_OK; }
      if (key == 4) {
        if (value > 160 * 1024) return fail(AKO_ERR_INVALID_ARGUMENT, "LDS reserve above 160 KiB");
        ako::g_rms_tuning.lds_reserve = value;
        return AKO_OK;
      }
      if (key == 5) {
        if (value > 2) return fail(AKO_ERR_INVALID_ARGUMENT, "row order must be 0, 1 or 2");
        ako::g_rms_tuning.row_order = value;
        return AKO_OK;
      }
      if (key == 6) { ako::g_rms_tuning.xcd_chunk = value; return AKO_OK; }
      if (key == 7) { ako::g_rms_tuning.max_blocks = value; return AKO_OK; }
      if (key == 8) {
        if (value > 2) return fail(AKO_ERR_INVALID_ARGUMENT, "early weights must be 0, 1 or 2");
        ako::g_rms_tuning.early_weights = value;
        return AKO_OK;
      }
      if (key == 9) {
        if (value > 2) return fail(AKO_ERR_INVALID_ARGUMENT, "pipeline must be 0, 1 or 2");
        ako::g_rms_tuning.pipeline = value;
        return AKO_OK;
      }
      if (key == 10) {
        if (value > 32) return fail(AKO_ERR_INVALID_ARGUMENT, "pipelined workgroups per CU above 32");
        ako::g_rms_tuning.pipe_blocks_per_cu = value;
        return AKO_OK;
      }
      if (key == 11) {
        if (value > 2) return fail(AKO_ERR_INVALID_ARGUMENT, "load groups must be 0, 1 or 2");
        ako::g_rms_tuning.load_groups = value;
        return AKO_OK;
      }
      if (key == 12) {
        if (value > 2) return fail(AKO_ERR_INVALID_ARGUMENT, "write-through stores must be 0, 1 or 2");
        ako::g_rms_tuning.write_through = value;
        return AKO_OK;
      }
      break;
    case 1:
      if (key == 1) { ako::g_rope_tuning.waves_per_block = value; return AKO_OK; }
      if (key == 2) return AKO_OK;  // head groups per wavefront, once: every lane moves one packet
      if (key == 3) { ako::g_rope_tuning.xcd_chunk = value; return AKO_OK; }
      break;
    case 2:
      if (key == 1) { ako::g_swiglu_tuning.vecs_per_thread = value; return AKO_OK; }
      if (key == 2) { ako::g_swiglu_tuning.xcd_chunk = value; return AKO_OK; }
      break;
    case 3:
      if (value > 65536) return fail(AKO_ERR_INVALID_ARGUMENT, "paged attention tuning values are at most 65536");
      if (key == 1) { ako::g_paged_tuning.items = value; return AKO_OK; }
      if (key == 2) { ako::g_paged_tuning.min_keys = value; return AKO_OK; }
      if (key == 3) {
        if (value > 2) return fail(AKO_ERR_INVALID_ARGUMENT, "paged attention kernel must be 0, 1 or 2, got %d", value);
        ako::g_paged_tuning.kernel = value;
        return AKO_OK;
      }
      break;
    default:
      break;
  }
  return fail(AKO_ERR_INVALID_ARGUMENT, "unknown tuning key op=%d key=%d", op, key);
}

// ---------------------------------------------------------------- RMSNorm --
static int rmsnorm_common(const void* x, const void* r, const void* w, void* y, void* rout,
                          int64_t rows, int64_t hidden, int64_t sx, int64_t sr, int64_t sy,
                          int64_t srout, float eps, int dtype, int w_dtype, void* stream,
                          bool residual) {
  const char* fn = residual ? "ako_rmsnorm_residual_fwd" : "ako_rmsnorm_fwd";
  if (!valid_dtype(dtype)) return fail(AKO_ERR_UNSUPPORTED, "%s: unknown dtype code %d", fn, dtype);
  if (w_dtype != dtype && w_dtype != AKO_DTYPE_F32)
    return fail(AKO_ERR_UNSUPPORTED, "%s: weight dtype %s with input dtype %s (weight must match or be f32)",
                fn, dtype_name(w_dtype), dtype_name(dtype));
  if (rows < 0 || hidden < 0) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: negative size rows=%lld hidden=%lld", fn, (long long)rows, (long long)hidden);
  if (rows == 0 || hidden == 0) return AKO_OK;
  if (hidden > kMaxInt) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: hidden=%lld exceeds 2^31-1", fn, (long long)hidden);
  if (!x || !w || !y || (residual && (!r || !rout)))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
  if (!(eps >= 0.0f)) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: eps must be >= 0", fn);
  if (sx < 0 || sy < 0 || (residual && (sr < 0 || srout < 0)))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: negative row stride", fn);
  if (rows > 1 && (sy < hidden || (residual && srout < hidden)))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: output row stride smaller than hidden (rows would overlap)", fn);
  const int eb = ako::dtype_bytes(dtype);
  const Span sy_span = span_2d(y, rows, hidden, sy, eb);
  const Span sx_span = span_2d(x, rows, hidden, sx, eb);
  const Span w_span = span_2d(w, 1, hidden, hidden, ako::dtype_bytes(w_dtype));
  if (!sy_span.ok || !sx_span.ok ||
      (residual && (!span_2d(r, rows, hidden, sr, eb).ok || !span_2d(rout, rows, hidden, srout, eb).ok)))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: sizes and strides overflow the address space", fn);
  if (overlap(sy_span, sx_span) || overlap(sy_span, w_span))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: output y overlaps an input", fn);
  if (residual) {
    const Span sr_span = span_2d(r, rows, hidden, sr, eb);
    const Span so_span = span_2d(rout, rows, hidden, srout, eb);
    if (overlap(sy_span, sr_span) || overlap(so_span, sx_span) || overlap(so_span, sr_span) ||
        overlap(so_span, w_span) || overlap(so_span, sy_span))
      return fail(AKO_ERR_INVALID_ARGUMENT, "%s: residual_out overlaps another buffer", fn);
  }
  bool aligned16 = aligned(x, 16) && aligned(y, 16) && aligned(w, 16) && (sx * eb) % 16 == 0 && (sy * eb) % 16 == 0;
  if (residual)
    aligned16 = aligned16 && aligned(r, 16) && aligned(rout, 16) && (sr * eb) % 16 == 0 && (srout * eb) % 16 == 0;
  ako::RmsArgs a{x, r, w, y, rout, rows, hidden, sx, sr, sy, srout, eps, dtype, w_dtype, residual, aligned16};
  return hip_status(ako::launch_rmsnorm(a, static_cast<hipStream_t>(stream)), fn);
}

int ako_rmsnorm_fwd(const void* x, const void* w, void* y, int64_t rows, int64_t hidden,
                    int64_t x_row_stride, int64_t y_row_stride, float eps, int dtype, int w_dtype,
                    void* stream) {
  return rmsnorm_common(x, nullptr, w, y, nullptr, rows, hidden, x_row_stride, 0, y_row_stride, 0,
                        eps, dtype, w_dtype, stream, false);
}

int ako_rmsnorm_residual_fwd(const void* x, const void* residual, const void* w, void* y,
                             void* residual_out, int64_t rows, int64_t hidden,
                             int64_t x_row_stride, int64_t r_row_stride, int64_t y_row_stride,
                             int64_t rout_row_stride, float eps, int dtype, int w_dtype,
                             void* stream) {
  return rmsnorm_common(x, residual, w, y, residual_out, rows, hidden, x_row_stride, r_row_stride,
                        y_row_stride, rout_row_stride, eps, dtype, w_dtype, stream, true);
}

// ------------------------------------------- RMSNorm over a sharded row --
int ako_rmsnorm_shard_partial_fwd(const void* x, const void* residual, void* residual_out,
                                  float* partial_ss, int64_t rows, int64_t shard,
                                  int64_t x_row_stride, int64_t r_row_stride,
                                  int64_t rout_row_stride, int dtype, void* stream) {
  const char* fn = "ako_rmsnorm_shard_partial_fwd";
  if (!valid_dtype(dtype)) return fail(AKO_ERR_UNSUPPORTED, "%s: unknown dtype code %d", fn, dtype);
  if (rows < 0 || shard < 0) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: negative size", fn);
  if (rows == 0) return AKO_OK;
  if (shard > kMaxInt) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: shard=%lld exceeds 2^31-1", fn, (long long)shard);
  const bool res = residual != nullptr;
  if ((residual == nullptr) != (residual_out == nullptr))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: residual and residual_out must both be given or both be null", fn);
  if (!partial_ss || (shard > 0 && !x)) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
  if (x_row_stride < 0 || (res && (r_row_stride < 0 || rout_row_stride < 0)))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: negative row stride", fn);
  if (res && rows > 1 && rout_row_stride < shard)
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: residual_out row stride smaller than the shard", fn);
  const int eb = ako::dtype_bytes(dtype);
  const Span ps = span_2d(partial_ss, 1, rows, rows, 4);
  const Span xs = span_2d(x, rows, shard, x_row_stride, eb);
  if (!ps.ok || !xs.ok) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: sizes and strides overflow the address space", fn);
  if (shard > 0 && overlap(ps, xs)) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: partial_ss overlaps x", fn);
  if (res) {
    const Span rs = span_2d(residual, rows, shard, r_row_stride, eb);
    const Span os = span_2d(residual_out, rows, shard, rout_row_stride, eb);
    if (!rs.ok || !os.ok) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: sizes and strides overflow the address space", fn);
    if (shard > 0 && (overlap(os, xs) || overlap(os, rs) || overlap(os, ps) || overlap(ps, rs)))
      return fail(AKO_ERR_INVALID_ARGUMENT, "%s: an output overlaps another buffer", fn);
  }
  ako::RmsShardArgs a{};
  a.x = x;
  a.r = residual;
  a.rout = residual_out;
  a.partial = partial_ss;
  a.rows = rows;
  a.shard = shard;
  a.sx = x_row_stride;
  a.sr = r_row_stride;
  a.srout = rout_row_stride;
  a.dtype = dtype;
  a.residual = res;
  return hip_status(ako::launch_rmsnorm_shard_partial(a, static_cast<hipStream_t>(stream)), fn);
}

int ako_rmsnorm_shard_apply_fwd(const void* s, const void* w, const float* total_ss, void* y,
                                int64_t rows, int64_t shard, int64_t hidden, int64_t s_row_stride,
                                int64_t y_row_stride, float eps, int dtype, int w_dtype,
                                void* stream) {
  const char* fn = "ako_rmsnorm_shard_apply_fwd";
  if (!valid_dtype(dtype)) return fail(AKO_ERR_UNSUPPORTED, "%s: unknown dtype code %d", fn, dtype);
  if (w_dtype != dtype && w_dtype != AKO_DTYPE_F32)
    return fail(AKO_ERR_UNSUPPORTED, "%s: weight dtype %s with input dtype %s (weight must match or be f32)",
                fn, dtype_name(w_dtype), dtype_name(dtype));
  if (rows < 0 || shard < 0 || hidden < 0) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: negative size", fn);
  if (rows == 0 || shard == 0) return AKO_OK;
  if (shard > hidden) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: shard %lld larger than hidden %lld", fn,
                                  (long long)shard, (long long)hidden);
  if (shard > kMaxInt) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: shard=%lld exceeds 2^31-1", fn, (long long)shard);
  if (!s || !w || !total_ss || !y) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
  if (!(eps >= 0.0f)) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: eps must be >= 0", fn);
  if (s_row_stride < 0 || y_row_stride < 0) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: negative row stride", fn);
  if (rows > 1 && y_row_stride < shard)
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: output row stride smaller than the shard", fn);
  const int eb = ako::dtype_bytes(dtype);
  const Span ss = span_2d(s, rows, shard, s_row_stride, eb);
  const Span ys = span_2d(y, rows, shard, y_row_stride, eb);
  const Span ws = span_2d(w, 1, shard, shard, ako::dtype_bytes(w_dtype));
  const Span ts = span_2d(total_ss, 1, rows, rows, 4);
  if (!ss.ok || !ys.ok || !ws.ok || !ts.ok)
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: sizes and strides overflow the address space", fn);
  if (overlap(ys, ss) || overlap(ys, ws) || overlap(ys, ts))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: output y overlaps an input", fn);
  ako::RmsShardArgs a{};
  a.x = s;
  a.w = w;
  a.total = total_ss;
  a.y = y;
  a.rows = rows;
  a.shard = shard;
  a.hidden = hidden;
  a.sx = s_row_stride;
  a.sy = y_row_stride;
  a.eps = eps;
  a.dtype = dtype;
  a.w_dtype = w_dtype;
  return hip_status(ako::launch_rmsnorm_shard_apply(a, static_cast<hipStream_t>(stream)), fn);
}

// ------------------------------------------------------------------- RoPE --
extern "C++" {  // C++ helpers inside the C-linkage block
namespace {

struct RopeTensorIn {
  const void* x;
  void* y;
  int64_t heads;
  const int64_t* xs;  // strides b, s, h
  const int64_t* ys;  // strides b, s (cache tensors: slot), h
  bool at_pos;        // output rows are cache slots (*pos + s), cache_len of them
};

// Byte span of a [n0, n1, n2, head_dim] view with the given element strides
// (last dimension contiguous): up to the last element + 1.
Span span_4d(const void* p, int64_t n0, int64_t n1, int64_t n2, int64_t d, const int64_t* st, int elem) {
  const __int128 last = static_cast<__int128>(n0 - 1) * st[0] + static_cast<__int128>(n1 - 1) * st[1] +
                        static_cast<__int128>(n2 - 1) * st[2] + d;
  return span_bytes(p, last * elem);
}

// True when distinct (i0, i1, i2, e) of a [n0, n1, n2, head_dim] view address
// distinct elements: taken in order of increasing stride, every dimension of
// more than one index must step past everything the smaller ones span. Any
// nesting order passes (heads-major cache slabs as well as token-major views).
bool distinct_rows(int64_t n0, int64_t n1, int64_t n2, int64_t head_dim, const int64_t* st) {
  struct Dim { int64_t stride, count; } dims[3] = {{st[0], n0}, {st[1], n1}, {st[2], n2}};
  for (int i = 0; i < 3; ++i)
    for (int j = i + 1; j < 3; ++j)
      if (dims[j].stride < dims[i].stride) std::swap(dims[i], dims[j]);
  __int128 reach = head_dim;
  for (const Dim& d : dims) {
    if (d.count <= 1) continue;
    if (d.stride < reach) return false;
    reach += static_cast<__int128>(d.stride) * (d.count - 1);
  }
  return true;
}

// Cache mode: pos != nullptr. Tensors with at_pos write rows 0..cache_len-1
// (selected on the device by *pos + s); the tables must hold table_rows >=
// cache_len rows. Tensor index 2 is copied, not rotated.
int rope_common(const char* fn, const RopeTensorIn* ts, int nt, const void* cos, const void* sin,
                int64_t batch, int64_t seq, int64_t head_dim, int64_t st, int dtype,
                int table_dtype, int style, void* stream, const int64_t* pos = nullptr,
                int64_t cache_len = 0, int64_t table_rows = 0) {
  if (!valid_dtype(dtype) || !valid_dtype(table_dtype))
    return fail(AKO_ERR_UNSUPPORTED, "%s: unknown dtype code (x %d, table %d)", fn, dtype, table_dtype);
  if (style != AKO_ROPE_NEOX && style != AKO_ROPE_INTERLEAVED)
    return fail(AKO_ERR_UNSUPPORTED, "%s: unknown RoPE style %d", fn, style);
  if (batch < 0 || seq < 0 || head_dim < 0)
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: negative size", fn);
  if (head_dim % 2 != 0) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: head_dim must be even, got %lld", fn, (long long)head_dim);
  const bool cache = pos != nullptr;
  if (cache && (cache_len <= 0 || cache_len > kMaxInt))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: cache_len must be in [1, 2^31-1], got %lld", fn, (long long)cache_len);
  if (cache && table_rows < cache_len)
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: the tables hold %lld rows, fewer than cache_len %lld", fn,
                (long long)table_rows, (long long)cache_len);
  int64_t total_heads = 0;
  for (int i = 0; i < nt; ++i) {
    if (ts[i].heads < 0) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: negative head count", fn);
    total_heads += ts[i].heads;
  }
  if (batch == 0 || seq == 0 || head_dim == 0 || total_heads == 0) return AKO_OK;
  if (head_dim > kMaxInt) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: head_dim too large", fn);
  if (batch > kMaxInt / seq || total_heads > kMaxInt)
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: batch*seq and the head count must stay below 2^31", fn);
  if (!cos || !sin) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: null table pointer", fn);
  const int64_t tab_rows = cache ? cache_len : seq;  // rows the kernel may read
  if (st < head_dim / 2 && tab_rows > 1) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: table row stride %lld < head_dim/2", fn, (long long)st);
  const int eb = ako::dtype_bytes(dtype);
  const int tb = ako::dtype_bytes(table_dtype);
  const Span cos_span = span_2d(cos, tab_rows, head_dim / 2, st, tb);
  const Span sin_span = span_2d(sin, tab_rows, head_dim / 2, st, tb);
  if (!cos_span.ok || !sin_span.ok)
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: table sizes and strides overflow the address space", fn);
  Span out_spans[3], in_spans[3];
  for (int i = 0; i < nt; ++i) {
    const RopeTensorIn& t = ts[i];
    if (t.heads == 0) continue;
    if (!t.x || !t.y || !t.xs || !t.ys) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: null tensor pointer", fn);
    for (int k = 0; k < 3; ++k)
      if (t.xs[k] < 0 || t.ys[k] < 0) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: negative stride", fn);
    const int64_t out_rows = t.at_pos ? cache_len : seq;
    // Distinct output elements must not alias.
    if (!distinct_rows(batch, out_rows, t.heads, head_dim, t.ys))
      return fail(AKO_ERR_INVALID_ARGUMENT, "%s: output strides make rows overlap", fn);
    in_spans[i] = span_4d(t.x, batch, seq, t.heads, head_dim, t.xs, eb);
    out_spans[i] = span_4d(t.y, batch, out_rows, t.heads, head_dim, t.ys, eb);
    if (!in_spans[i].ok || !out_spans[i].ok)
      return fail(AKO_ERR_INVALID_ARGUMENT, "%s: sizes and strides overflow the address space", fn);
  }
  if (cache) {
    const Span pos_span{reinterpret_cast<uintptr_t>(pos), reinterpret_cast<uintptr_t>(pos) + sizeof(int64_t)};
    for (int i = 0; i < nt; ++i)
      if (ts[i].heads != 0 && overlap(out_spans[i], pos_span))
        return fail(AKO_ERR_INVALID_ARGUMENT, "%s: an output overlaps pos", fn);
  }
  for (int i = 0; i < nt; ++i) {
    if (ts[i].heads == 0) continue;
    if (overlap(out_spans[i], cos_span) || overlap(out_spans[i], sin_span))
      return fail(AKO_ERR_INVALID_ARGUMENT, "%s: output overlaps a table", fn);
    for (int k = 0; k < nt; ++k) {
      if (ts[k].heads == 0) continue;
      if (overlap(out_spans[i], in_spans[k]))
        return fail(AKO_ERR_INVALID_ARGUMENT, "%s: output overlaps an input", fn);
      if (k != i && overlap(out_spans[i], out_spans[k]))
        return fail(AKO_ERR_INVALID_ARGUMENT, "%s: two outputs overlap", fn);
    }
  }

  ako::RopeArgs a{};
  const ako::RopeTensorArgs none{nullptr, nullptr, 0, 0, 0, 0, 0, 0, 0};
  auto conv = [&](const RopeTensorIn& t) {
    if (t.heads == 0) return none;
    return ako::RopeTensorArgs{t.x, t.y, t.heads, t.xs[0], t.xs[1], t.xs[2], t.ys[0], t.ys[1], t.ys[2]};
  };
  a.t0 = conv(ts[0]);
  a.t1 = nt > 1 ? conv(ts[1]) : none;
  a.t2 = nt > 2 ? conv(ts[2]) : none;
  // Without a cache the roles of t0 and t1 are the same; a launch with only
  // the second tensor moves it first. In cache mode the roles differ (t0 is
  // written at s, t1 at the cache slot) and an empty t0 simply has no heads.
  if (!cache && a.t0.heads == 0) { a.t0 = a.t1; a.t1 = none; }
  a.pos = pos;
  a.cache_len = cache ? cache_len : 0;
  a.cos = cos;
  a.sin = sin;
  a.batch = batch;
  a.seq = seq;
  a.head_dim = head_dim;
  a.st = st;
  a.dtype = dtype;
  a.table_dtype = table_dtype;
  a.neox = style == AKO_ROPE_NEOX;
  return hip_status(ako::launch_rope(a, static_cast<hipStream_t>(stream)), fn);
}

}  // namespace
}  // extern "C++"

int ako_rope_fwd(const void* x, const void* cos_table, const void* sin_table, void* y,
                 int64_t batch, int64_t seq, int64_t heads, int64_t head_dim, int64_t x_stride_b,
                 int64_t x_stride_s, int64_t x_stride_h, int64_t y_stride_b, int64_t y_stride_s,
                 int64_t y_stride_h, int64_t table_row_stride, int dtype, int table_dtype,
                 int style, void* stream) {
  const int64_t xs[3] = {x_stride_b, x_stride_s, x_stride_h};
  const int64_t ys[3] = {y_stride_b, y_stride_s, y_stride_h};
  const RopeTensorIn t{x, y, heads, xs, ys, false};
  return rope_common("ako_rope_fwd", &t, 1, cos_table, sin_table, batch, seq, head_dim,
                     table_row_stride, dtype, table_dtype, style, stream);
}

int ako_rope_qk_fwd(const void* q, const void* k, const void* cos_table, const void* sin_table,
                    void* q_out, void* k_out, int64_t batch, int64_t seq, int64_t q_heads,
                    int64_t k_heads, int64_t head_dim, const int64_t* q_strides,
                    const int64_t* k_strides, const int64_t* q_out_strides,
                    const int64_t* k_out_strides, int64_t table_row_stride, int dtype,
                    int table_dtype, int style, void* stream) {
  const RopeTensorIn ts[2] = {{q, q_out, q_heads, q_strides, q_out_strides, false},
                              {k, k_out, k_heads, k_strides, k_out_strides, false}};
  return rope_common("ako_rope_qk_fwd", ts, 2, cos_table, sin_table, batch, seq, head_dim,
                     table_row_stride, dtype, table_dtype, style, stream);
}

int ako_rope_qk_cache_fwd(const void* q, const void* k, const void* v, const void* cos_table,
                          const void* sin_table, void* q_out, void* k_cache, void* v_cache,
                          const int64_t* pos, int64_t batch, int64_t seq, int64_t q_heads,
                          int64_t kv_heads, int64_t head_dim, const int64_t* q_strides,
                          const int64_t* k_strides, const int64_t* v_strides,
                          const int64_t* q_out_strides, const int64_t* cache_strides,
                          int64_t cache_len, int64_t table_rows, int64_t table_row_stride,
                          int dtype, int table_dtype, int style, void* stream) {
  const char* fn = "ako_rope_qk_cache_fwd";
  if (!pos) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: null pos pointer", fn);
  if ((v == nullptr) != (v_cache == nullptr))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: v and v_cache must both be given or both be null", fn);
  const int64_t v_heads = v ? kv_heads : 0;
  const RopeTensorIn ts[3] = {{q, q_out, q_heads, q_strides, q_out_strides, false},
                              {k, k_cache, kv_heads, k_strides, cache_strides, true},
                              {v, v_cache, v_heads, v_strides, cache_strides, true}};
  return rope_common(fn, ts, 3, cos_table, sin_table, batch, seq, head_dim, table_row_stride, dtype,
                     table_dtype, style, stream, pos, cache_len, table_rows);
}

// ----------------------------------------------------------------- SwiGLU --
int ako_swiglu_fwd(const void* gate, const void* up, void* y, int64_t rows, int64_t n,
                   int64_t gate_row_stride, int64_t up_row_stride, int64_t y_row_stride,
                   int dtype, void* stream) {
  const char* fn = "ako_swiglu_fwd";
  if (!valid_dtype(dtype)) return fail(AKO_ERR_UNSUPPORTED, "%s: unknown dtype code %d", fn, dtype);
  if (rows < 0 || n < 0) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: negative size", fn);
  if (rows == 0 || n == 0) return AKO_OK;
  if (n > kMaxInt) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: n=%lld exceeds 2^31-1", fn, (long long)n);
  if (!gate || !up || !y) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
  if (gate_row_stride < 0 || up_row_stride < 0 || y_row_stride < 0)
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: negative row stride", fn);
  if (rows > 1 && y_row_stride < n)
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: output row stride smaller than n (rows would overlap)", fn);
  const int eb = ako::dtype_bytes(dtype);
  const Span ys = span_2d(y, rows, n, y_row_stride, eb);
  const Span gs = span_2d(gate, rows, n, gate_row_stride, eb);
  const Span us = span_2d(up, rows, n, up_row_stride, eb);
  if (!ys.ok || !gs.ok || !us.ok)
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: sizes and strides overflow the address space", fn);
  if (overlap(ys, gs) || overlap(ys, us))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: output overlaps an input", fn);
  const bool contiguous = rows == 1 || (gate_row_stride == n && up_row_stride == n && y_row_stride == n);
  ako::SwigluArgs a{gate, up, y, rows, n, gate_row_stride, up_row_stride, y_row_stride, dtype, contiguous};
  return hip_status(ako::launch_swiglu(a, static_cast<hipStream_t>(stream)), fn);
}

// ------------------------------------------------- paged key/value cache --
extern "C++" {
namespace {

// Positions are 32-bit, with room for a tile past the last one.
constexpr int64_t kMaxPositions = kMaxInt - 65536;

bool valid_page_dtype(int page_dtype, int dtype) { return page_dtype == dtype || page_dtype == AKO_DTYPE_E4M3; }

// Checks what every call over a paged cache needs and fills the launchers'
// arguments. `empty` is set when there are no rows: the call is then done.
int paged_common(const char* fn, const ako_paged_t* c, int64_t heads, int dtype, ako::PagedArgs* out, bool* empty) {
  if (!c) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: null cache", fn);
  if (!valid_dtype(dtype)) return fail(AKO_ERR_UNSUPPORTED, "%s: unknown dtype code %d", fn, dtype);
  if (!valid_page_dtype(c->page_dtype, dtype))
    return fail(AKO_ERR_UNSUPPORTED, "%s: pages of dtype code %d for rows of %s", fn, c->page_dtype, dtype_name(dtype));
  if (c->num_pages < 0 || c->n_seqs < 0 || c->table_width < 0 || c->tokens < 0 || heads < 0)
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: negative size", fn);
  if (c->head_dim < 16 || c->head_dim > 256 || c->head_dim % 16)
    return fail(AKO_ERR_UNSUPPORTED, "%s: head_dim must be a multiple of 16 up to 256, got %lld", fn, (long long)c->head_dim);
  if (c->kv_heads < 1 || c->page_size < 1)
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: kv_heads and page_size must be at least 1", fn);
  if (c->page_size > kMaxPositions || c->table_width > kMaxPositions / c->page_size)
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: the block table names 2^31-65537 positions or more", fn);
  if (c->kv_heads > kMaxInt / 65536 || heads > kMaxInt / 65536 || c->num_pages > kMaxInt || c->n_seqs > kMaxInt / 2 ||
      c->tokens > kMaxInt / 2 / std::max<int64_t>(1, std::max(heads, c->kv_heads)))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: too many heads, pages, sequences or rows", fn);
  if (!c->cu_seqlens && c->tokens > 0 && (c->n_seqs == 0 || c->tokens % c->n_seqs))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: %lld rows are no multiple of %lld sequences", fn, (long long)c->tokens,
                (long long)c->n_seqs);
  *empty = c->tokens == 0;
  const bool mx = c->page_dtype == AKO_DTYPE_E4M3;
  for (int i = 0; i < 3; ++i)
    if (c->k_strides[i] < 0 || c->v_strides[i] < 0 || (mx && (c->k_scale_strides[i] < 0 || c->v_scale_strides[i] < 0)))
      return fail(AKO_ERR_INVALID_ARGUMENT, "%s: negative page stride", fn);
  if (c->table_stride < 0 || (c->table_stride < c->table_width && c->n_seqs > 1))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: block table rows overlap", fn);
  if (*empty) return AKO_OK;
  if (c->num_pages > 0 && (!c->k_pages || !c->v_pages || (mx && (!c->k_scales || !c->v_scales))))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: null pages or scales", fn);
  if (!mx && (c->k_scales || c->v_scales))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: scales are for e4m3 pages", fn);
  if (c->n_seqs > 0 && (!c->seq_lens || (c->table_width > 0 && !c->block_table)))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: null block table or lengths", fn);
  ako::PagedArgs& a = *out;
  a.k = c->k_pages;
  a.v = c->v_pages;
  a.ks = c->k_scales;
  a.vs = c->v_scales;
  a.mx = mx;
  a.table = c->block_table;
  a.lens = c->seq_lens;
  a.cu = c->cu_seqlens;
  for (int i = 0; i < 3; ++i) {
    a.kst[i] = c->k_strides[i];
    a.vst[i] = c->v_strides[i];
    a.ksst[i] = mx ? c->k_scale_strides[i] : 0;
    a.vsst[i] = mx ? c->v_scale_strides[i] : 0;
  }
  a.table_stride = c->table_stride;
  a.table_width = c->table_width;
  a.n_seqs = c->n_seqs;
  a.num_pages = c->num_pages;
  a.kv_heads = c->kv_heads;
  a.page_size = c->page_size;
  a.head_dim = c->head_dim;
  a.tokens = c->tokens;
  return AKO_OK;
}

// The memory a cache call reads or writes: pages and scales, then the step's
// own index tensors.
struct PagedSpans {
  Span pages[4], index[3];
  int n_pages = 0, n_index = 0;
  bool ok = true;

  PagedSpans(const ako_paged_t* c, int dtype) {
    const bool mx = c->page_dtype == AKO_DTYPE_E4M3;
    const int eb = mx ? 1 : ako::dtype_bytes(dtype);
    const int64_t codes = ako::ceil_div(c->head_dim, 32);
    if (c->num_pages > 0) {
      add(span_4d(c->k_pages, c->num_pages, c->kv_heads, c->page_size, c->head_dim, c->k_strides, eb));
      add(span_4d(c->v_pages, c->num_pages, c->kv_heads, c->page_size, c->head_dim, c->v_strides, eb));
      if (mx) {
        add(span_4d(c->k_scales, c->num_pages, c->kv_heads, c->page_size, codes, c->k_scale_strides, 1));
        add(span_4d(c->v_scales, c->num_pages, c->kv_heads, c->page_size, codes, c->v_scale_strides, 1));
      }
    }
    if (c->n_seqs > 0) {
      if (c->table_width > 0) add_index(span_2d(c->block_table, c->n_seqs, c->table_width, c->table_stride, 4));
      add_index(span_2d(c->seq_lens, 1, c->n_seqs, c->n_seqs, 4));
    }
    if (c->cu_seqlens) add_index(span_2d(c->cu_seqlens, 1, c->n_seqs + 1, c->n_seqs + 1, 4));
  }
  bool meets(const Span& s) const {
    for (int i = 0; i < n_pages; ++i)
      if (overlap(pages[i], s)) return true;
    return meets_index(s);
  }
  bool meets_index(const Span& s) const {
    for (int i = 0; i < n_index; ++i)
      if (overlap(index[i], s)) return true;
    return false;
  }

 private:
  void add(const Span& s) {
    ok = ok && s.ok;
    pages[n_pages++] = s;
  }
  void add_index(const Span& s) {
    ok = ok && s.ok;
    index[n_index++] = s;
  }
};

// Whether rows of `width` bytes at a and at b (same shape and strides, in
// bytes) never share a byte: apart altogether, or interleaved in one
// allocation with every row of one between rows of the other.
bool rows_apart(const Span& sa, const Span& sb, int64_t n0, int64_t n1, int64_t n2, int64_t width, const int64_t* st_a,
                const int64_t* st_b, int eb) {
  if (!overlap(sa, sb)) return true;
  for (int i = 0; i < 3; ++i)
    if (st_a[i] != st_b[i]) return false;
  const uint64_t gap = sa.lo < sb.lo ? sb.lo - sa.lo : sa.lo - sb.lo;
  struct Dim { __int128 stride; int64_t count; } dims[4] = {
      {__int128(st_a[0]) * eb, n0}, {__int128(st_a[1]) * eb, n1}, {__int128(st_a[2]) * eb, n2}, {__int128(gap), 2}};
  for (int i = 0; i < 4; ++i)
    for (int j = i + 1; j < 4; ++j)
      if (dims[j].stride < dims[i].stride) std::swap(dims[i], dims[j]);
  __int128 reach = __int128(width) * eb;
  for (const Dim& d : dims) {
    if (d.count <= 1) continue;
    if (d.stride < reach) return false;
    reach += d.stride * (d.count - 1);
  }
  return true;
}

}  // namespace
}  // extern "C++"

extern "C++" {
namespace {

// RMSNorm weights of a call's heads; no weights: no norm.
struct HeadNorm {
  const void* qw = nullptr;
  const void* kw = nullptr;
  float eps = 0.0f;
  int w_dtype = 0;
};

int norm_args(const char* fn, const HeadNorm& w, int dtype) {
  if (w.w_dtype != dtype && w.w_dtype != AKO_DTYPE_F32)
    return fail(AKO_ERR_UNSUPPORTED, "%s: weight dtype %s with input dtype %s (weight must match or be f32)", fn,
                dtype_name(w.w_dtype), dtype_name(dtype));
  if (!(w.eps >= 0.0f)) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: eps must be >= 0", fn);
  return AKO_OK;
}

int paged_write(const char* fn, const HeadNorm* norm, const void* q, const void* k, const void* v, const void* cos_table,
                const void* sin_table, void* q_out, const ako_paged_t* cache, int64_t q_heads, const int64_t* q_strides,
                const int64_t* k_strides, const int64_t* v_strides, int64_t table_rows, int64_t table_row_stride, int dtype,
                int table_dtype, int style, void* stream) {
  ako::PagedWriteArgs a{};
  bool empty = false;
  if (const int rc = paged_common(fn, cache, q_heads, dtype, &a.c, &empty)) return rc;
  if (!valid_dtype(table_dtype)) return fail(AKO_ERR_UNSUPPORTED, "%s: unknown table dtype code %d", fn, table_dtype);
  if (style != AKO_ROPE_NEOX && style != AKO_ROPE_INTERLEAVED)
    return fail(AKO_ERR_UNSUPPORTED, "%s: unknown RoPE style %d", fn, style);
  if (table_rows < 0) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: negative size", fn);
  if (norm)
    if (const int rc = norm_args(fn, *norm, dtype)) return rc;
  if (empty) return AKO_OK;
  const int64_t d = cache->head_dim, kvh = cache->kv_heads, n = cache->num_pages, ps = cache->page_size;
  const int64_t per = cache->cu_seqlens ? cache->tokens : cache->tokens / cache->n_seqs;
  const int64_t seqs = cache->cu_seqlens ? 1 : cache->n_seqs;
  if ((q_heads > 0 && (!q || !q_out)) || !k || !v || !q_strides || !k_strides || !v_strides ||
      (table_rows > 0 && (!cos_table || !sin_table)))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
  if (table_row_stride < 0 || (table_rows > 1 && table_row_stride < d / 2))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: table row stride %lld < head_dim/2", fn, (long long)table_row_stride);
  for (int i = 0; i < 3; ++i)
    if (q_strides[i] < 0 || k_strides[i] < 0 || v_strides[i] < 0)
      return fail(AKO_ERR_INVALID_ARGUMENT, "%s: negative stride", fn);
  const int eb = ako::dtype_bytes(dtype), tb = ako::dtype_bytes(table_dtype);
  const PagedSpans held(cache, dtype);
  Span in[7];
  int n_in = 0;
  if (norm) {
    if (!norm->qw || !norm->kw) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: null weight", fn);
    const int wb = ako::dtype_bytes(norm->w_dtype);
    in[n_in++] = span_2d(norm->qw, 1, d, d, wb);
    in[n_in++] = span_2d(norm->kw, 1, d, d, wb);
    a.qw = norm->qw;
    a.kw = norm->kw;
    a.eps = norm->eps;
    a.w_dtype = norm->w_dtype;
  }
  if (q_heads > 0) in[n_in++] = span_4d(q, seqs, per, q_heads, d, q_strides, eb);
  in[n_in++] = span_4d(k, seqs, per, kvh, d, k_strides, eb);
  in[n_in++] = span_4d(v, seqs, per, kvh, d, v_strides, eb);
  if (table_rows > 0) {
    in[n_in++] = span_2d(cos_table, table_rows, d / 2, table_row_stride, tb);
    in[n_in++] = span_2d(sin_table, table_rows, d / 2, table_row_stride, tb);
  }
  const Span qo = span_2d(q_out, 1, cache->tokens * q_heads * d, 0, eb);
  bool ok = held.ok && qo.ok;
  for (int i = 0; i < n_in; ++i) ok = ok && in[i].ok;
  if (!ok) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: sizes and strides overflow the address space", fn);
  for (int i = 0; i < n_in; ++i) {
    if (q_heads > 0 && overlap(qo, in[i])) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: q_out overlaps an input", fn);
    for (int j = 0; j < held.n_pages; ++j)
      if (overlap(held.pages[j], in[i])) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: the pages overlap an input", fn);
  }
  if (q_heads > 0 && held.meets(qo))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: q_out overlaps the cache or its indexes", fn);
  for (int j = 0; j < held.n_pages; ++j)
    if (held.meets_index(held.pages[j]))
      return fail(AKO_ERR_INVALID_ARGUMENT, "%s: the pages overlap the block table or the lengths", fn);
  if (n > 0) {
    const bool mx = cache->page_dtype == AKO_DTYPE_E4M3;
    const int pb = mx ? 1 : eb;
    const int64_t codes = ako::ceil_div(d, 32);
    bool apart = distinct_rows(n, kvh, ps, d, cache->k_strides) && distinct_rows(n, kvh, ps, d, cache->v_strides) &&
                 rows_apart(held.pages[0], held.pages[1], n, kvh, ps, d, cache->k_strides, cache->v_strides, pb);
    if (mx)
      apart = apart && distinct_rows(n, kvh, ps, codes, cache->k_scale_strides) &&
              distinct_rows(n, kvh, ps, codes, cache->v_scale_strides) &&
              rows_apart(held.pages[2], held.pages[3], n, kvh, ps, codes, cache->k_scale_strides, cache->v_scale_strides, 1) &&
              !overlap(held.pages[0], held.pages[2]) && !overlap(held.pages[0], held.pages[3]) &&
              !overlap(held.pages[1], held.pages[2]) && !overlap(held.pages[1], held.pages[3]);
    if (!apart) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: rows of the cache overlap", fn);
  }
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_out = q_out;
  a.cos = cos_table;
  a.sin = sin_table;
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = q_strides[i];
    a.kns[i] = k_strides[i];
    a.vns[i] = v_strides[i];
  }
  a.st = table_row_stride;
  a.table_rows = table_rows;
  a.q_heads = q_heads;
  a.dtype = dtype;
  a.table_dtype = table_dtype;
  a.neox = style == AKO_ROPE_NEOX;
  return hip_status(ako::launch_paged_write(a, static_cast<hipStream_t>(stream)), fn);
}

}  // namespace
}  // extern "C++"

int ako_rope_qk_paged_fwd(const void* q, const void* k, const void* v, const void* cos_table, const void* sin_table,
                          void* q_out, const ako_paged_t* cache, int64_t q_heads, const int64_t* q_strides,
                          const int64_t* k_strides, const int64_t* v_strides, int64_t table_rows,
                          int64_t table_row_stride, int dtype, int table_dtype, int style, void* stream) {
  return paged_write("ako_rope_qk_paged_fwd", nullptr, q, k, v, cos_table, sin_table, q_out, cache, q_heads, q_strides,
                     k_strides, v_strides, table_rows, table_row_stride, dtype, table_dtype, style, stream);
}

int ako_rmsnorm_rope_qk_paged_fwd(const void* q, const void* k, const void* v, const void* q_weight, const void* k_weight,
                                  const void* cos_table, const void* sin_table, void* q_out, const ako_paged_t* cache,
                                  int64_t q_heads, const int64_t* q_strides, const int64_t* k_strides,
                                  const int64_t* v_strides, int64_t table_rows, int64_t table_row_stride, float eps,
                                  int dtype, int w_dtype, int table_dtype, int style, void* stream) {
  const HeadNorm norm{q_weight, k_weight, eps, w_dtype};
  return paged_write("ako_rmsnorm_rope_qk_paged_fwd", &norm, q, k, v, cos_table, sin_table, q_out, cache, q_heads, q_strides,
                     k_strides, v_strides, table_rows, table_row_stride, dtype, table_dtype, style, stream);
}

int ako_rmsnorm_rope_qk_fwd(const void* q, const void* k, const void* q_weight, const void* k_weight,
                            const void* cos_table, const void* sin_table, void* q_out, void* k_out, int64_t batch,
                            int64_t seq, int64_t q_heads, int64_t k_heads, int64_t head_dim, const int64_t* q_strides,
                            const int64_t* k_strides, int64_t table_row_stride, float eps, int dtype, int w_dtype,
                            int table_dtype, int style, void* stream) {
  const char* fn = "ako_rmsnorm_rope_qk_fwd";
  if (!valid_dtype(dtype) || !valid_dtype(table_dtype))
    return fail(AKO_ERR_UNSUPPORTED, "%s: unknown dtype code (x %d, table %d)", fn, dtype, table_dtype);
  if (style != AKO_ROPE_NEOX && style != AKO_ROPE_INTERLEAVED)
    return fail(AKO_ERR_UNSUPPORTED, "%s: unknown RoPE style %d", fn, style);
  const HeadNorm norm{q_weight, k_weight, eps, w_dtype};
  if (const int rc = norm_args(fn, norm, dtype)) return rc;
  if (batch < 0 || seq < 0 || q_heads < 0 || k_heads < 0) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: negative size", fn);
  if (head_dim < 2 || head_dim > 512 || head_dim % 2)
    return fail(AKO_ERR_UNSUPPORTED, "%s: head_dim must be even and 2 to 512, got %lld", fn, (long long)head_dim);
  if (batch == 0 || seq == 0 || (q_heads == 0 && k_heads == 0)) return AKO_OK;
  constexpr int64_t kMaxHeads = int64_t(1) << 23;  // of q or of k: a token's lanes stay below 2^30
  if (batch > kMaxInt / seq || q_heads > kMaxHeads || k_heads > kMaxHeads)
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: batch*seq must stay below 2^31, the heads at most 2^23", fn);
  if ((q_heads > 0 && (!q || !q_out || !q_weight || !q_strides)) || (k_heads > 0 && (!k || !k_out || !k_weight || !k_strides)) ||
      !cos_table || !sin_table)
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
  if (table_row_stride < 0 || (seq > 1 && table_row_stride < head_dim / 2))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: table row stride %lld < head_dim/2", fn, (long long)table_row_stride);
  for (int i = 0; i < 3; ++i)
    if ((q_heads > 0 && q_strides[i] < 0) || (k_heads > 0 && k_strides[i] < 0))
      return fail(AKO_ERR_INVALID_ARGUMENT, "%s: negative stride", fn);
  const int eb = ako::dtype_bytes(dtype), tb = ako::dtype_bytes(table_dtype), wb = ako::dtype_bytes(w_dtype);
  const __int128 row = static_cast<__int128>(batch) * seq * head_dim * eb;
  Span in[6], out[2];
  int n_in = 0, n_out = 0;
  in[n_in++] = span_2d(cos_table, seq, head_dim / 2, table_row_stride, tb);
  in[n_in++] = span_2d(sin_table, seq, head_dim / 2, table_row_stride, tb);
  if (q_heads > 0) {
    in[n_in++] = span_4d(q, batch, seq, q_heads, head_dim, q_strides, eb);
    in[n_in++] = span_2d(q_weight, 1, head_dim, head_dim, wb);
    out[n_out++] = span_bytes(q_out, row * q_heads);
  }
  if (k_heads > 0) {
    in[n_in++] = span_4d(k, batch, seq, k_heads, head_dim, k_strides, eb);
    in[n_in++] = span_2d(k_weight, 1, head_dim, head_dim, wb);
    out[n_out++] = span_bytes(k_out, row * k_heads);
  }
  bool ok = true, apart = n_out < 2 || !overlap(out[0], out[1]);
  for (int i = 0; i < n_in; ++i) ok = ok && in[i].ok;
  for (int o = 0; o < n_out; ++o) {
    ok = ok && out[o].ok;
    for (int i = 0; i < n_in; ++i) apart = apart && !overlap(out[o], in[i]);
  }
  if (!ok) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: sizes and strides overflow the address space", fn);
  if (!apart) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: an output overlaps another buffer", fn);
  ako::NormRopeArgs a{};
  a.q = q;
  a.k = k;
  a.qw = q_weight;
  a.kw = k_weight;
  a.cos = cos_table;
  a.sin = sin_table;
  a.q_out = q_out;
  a.k_out = k_out;
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = q_heads > 0 ? q_strides[i] : 0;
    a.ks[i] = k_heads > 0 ? k_strides[i] : 0;
  }
  a.batch = batch;
  a.seq = seq;
  a.q_heads = q_heads;
  a.k_heads = k_heads;
  a.head_dim = head_dim;
  a.st = table_row_stride;
  a.eps = eps;
  a.dtype = dtype;
  a.w_dtype = w_dtype;
  a.table_dtype = table_dtype;
  a.neox = style == AKO_ROPE_NEOX;
  return hip_status(ako::launch_norm_rope(a, static_cast<hipStream_t>(stream)), fn);
}

int ako_paged_read_fwd(const ako_paged_t* cache, void* k_out, void* v_out, int dtype, void* stream) {
  const char* fn = "ako_paged_read_fwd";
  ako::PagedReadArgs a{};
  bool empty = false;
  if (const int rc = paged_common(fn, cache, 0, dtype, &a.c, &empty)) return rc;
  if (empty) return AKO_OK;
  if (!k_out || !v_out) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
  const int64_t n = cache->tokens * cache->kv_heads * cache->head_dim;
  const Span ko = span_2d(k_out, 1, n, 0, ako::dtype_bytes(dtype)), vo = span_2d(v_out, 1, n, 0, ako::dtype_bytes(dtype));
  const PagedSpans held(cache, dtype);
  if (!ko.ok || !vo.ok || !held.ok)
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: sizes and strides overflow the address space", fn);
  if (overlap(ko, vo) || held.meets(ko) || held.meets(vo))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: an output overlaps another buffer", fn);
  a.k_out = k_out;
  a.v_out = v_out;
  a.dtype = dtype;
  return hip_status(ako::launch_paged_read(a, static_cast<hipStream_t>(stream)), fn);
}

extern "C++" {
namespace {

int attention_common(const char* fn, const ako_paged_t* cache, int64_t q_heads, int dtype, ako::PagedAttentionArgs* a,
                     bool* empty) {
  if (const int rc = paged_common(fn, cache, q_heads, dtype, &a->c, empty)) return rc;
  if (q_heads % cache->kv_heads)
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: %lld query heads are no multiple of %lld", fn, (long long)q_heads,
                (long long)cache->kv_heads);
  *empty = *empty || q_heads == 0;
  a->q_heads = q_heads;
  a->dtype = dtype;
  a->tuned_items = ako::g_paged_tuning.items;
  a->tuned_min_keys = ako::g_paged_tuning.min_keys;
  a->tuned_kernel = ako::g_paged_tuning.kernel;
  return AKO_OK;
}

}  // namespace
}  // extern "C++"

extern "C++" {
namespace {

// `blocks`: those listed for each row and key head, `count` of them; 0: all.
int attend(const char* fn, const void* q, const int64_t* q_strides, void* out, const ako_paged_t* cache, int64_t q_heads,
           float scale, int64_t window, int64_t sinks, const int32_t* blocks, int64_t count, void* workspace,
           int64_t workspace_bytes, int dtype, void* stream) {
  ako::PagedAttentionArgs a{};
  bool empty = false;
  if (const int rc = attention_common(fn, cache, q_heads, dtype, &a, &empty)) return rc;
  if (!(scale - scale == 0.0f)) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: scale must be finite", fn);
  if (window < 0 || sinks < 0) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: window and sinks must be >= 0", fn);
  if (empty) return AKO_OK;
  if (!q || !out || !q_strides) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
  if (q_strides[0] < 0 || q_strides[1] < 0 || q_strides[2] < 0)
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: negative stride", fn);
  if (count > 0 && !blocks) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: null blocks", fn);
  a.window = window;
  a.sinks = sinks;
  a.blocks = blocks;
  a.block_count = count;
  const int64_t need = ako::paged_attention_workspace(a);
  if (workspace_bytes < need || (need > 0 && (!workspace || !aligned(workspace, 16))))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: needs a 16-byte aligned workspace of %lld bytes, got %lld", fn,
                (long long)need, (long long)workspace_bytes);
  const int64_t d = cache->head_dim;
  const int64_t per = cache->cu_seqlens ? cache->tokens : cache->tokens / cache->n_seqs;
  const Span qi = span_4d(q, cache->cu_seqlens ? 1 : cache->n_seqs, per, q_heads, d, q_strides, ako::dtype_bytes(dtype));
  const Span o = span_2d(out, 1, cache->tokens * q_heads * d, 0, ako::dtype_bytes(dtype));
  const Span w = span_bytes(workspace, need);
  const Span b = span_bytes(blocks, static_cast<__int128>(cache->tokens) * cache->kv_heads * count * 4);
  const PagedSpans held(cache, dtype);
  if (!qi.ok || !o.ok || !w.ok || !b.ok || !held.ok)
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: sizes and strides overflow the address space", fn);
  if (overlap(o, qi) || held.meets(o) || (count > 0 && overlap(o, b))) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: out overlaps an input", fn);
  if (overlap(w, qi) || overlap(w, o) || held.meets(w) || (count > 0 && overlap(w, b)))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: the workspace overlaps another buffer", fn);
  a.q = q;
  a.out = out;
  for (int i = 0; i < 3; ++i) a.qs[i] = q_strides[i];
  a.scale = scale;
  a.workspace = workspace;
  return hip_status(ako::launch_paged_attention(a, static_cast<hipStream_t>(stream)), fn);
}

}  // namespace
}  // extern "C++"

int ako_paged_attention_fwd(const void* q, const int64_t* q_strides, void* out, const ako_paged_t* cache, int64_t q_heads,
                            float scale, int64_t window, int64_t sinks, void* workspace, int64_t workspace_bytes, int dtype,
                            void* stream) {
  return attend("ako_paged_attention_fwd", q, q_strides, out, cache, q_heads, scale, window, sinks, nullptr, 0, workspace,
                workspace_bytes, dtype, stream);
}

int ako_paged_attention_blocks_fwd(const void* q, const int64_t* q_strides, void* out, const ako_paged_t* cache,
                                   int64_t q_heads, float scale, const int32_t* blocks, int64_t count, void* workspace,
                                   int64_t workspace_bytes, int dtype, void* stream) {
  const char* fn = "ako_paged_attention_blocks_fwd";
  if (count < 1 || count > kMaxInt / 2) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: count must be 1 to 2^30", fn);
  return attend(fn, q, q_strides, out, cache, q_heads, scale, 0, 0, blocks, count, workspace, workspace_bytes, dtype, stream);
}

int64_t ako_paged_attention_blocks_workspace(const ako_paged_t* cache, int64_t q_heads, int64_t count, int dtype) {
  const char* fn = "ako_paged_attention_blocks_workspace";
  ako::PagedAttentionArgs a{};
  bool empty = false;
  if (count < 1 || count > kMaxInt / 2) {
    fail(AKO_ERR_INVALID_ARGUMENT, "%s: count must be 1 to 2^30", fn);
    return -1;
  }
  if (attention_common(fn, cache, q_heads, dtype, &a, &empty)) return -1;
  a.block_count = count;
  return empty ? 0 : ako::paged_attention_workspace(a);
}

int64_t ako_paged_attention_workspace(const ako_paged_t* cache, int64_t q_heads, int dtype) {
  ako::PagedAttentionArgs a{};
  bool empty = false;
  if (attention_common("ako_paged_attention_workspace", cache, q_heads, dtype, &a, &empty)) return -1;
  return empty ? 0 : ako::paged_attention_workspace(a);
}

// ------------------------------------------------- blocks of a paged cache --
extern "C++" {
namespace {

// What a call on means has of a cache: the keys alone, or no pages at all.
ako_paged_t keys_only(const ako_paged_t& c) {
  ako_paged_t k = c;
  k.v_pages = c.k_pages;
  k.v_scales = c.k_scales;
  for (int i = 0; i < 3; ++i) {
    k.v_strides[i] = c.k_strides[i];
    k.v_scale_strides[i] = c.k_scale_strides[i];
  }
  return k;
}
ako_paged_t no_pages(const ako_paged_t& c, const void* means, int dtype) {
  ako_paged_t k = c;
  k.k_pages = const_cast<void*>(means);  // not read
  k.k_scales = nullptr;
  for (int i = 0; i < 3; ++i) k.k_strides[i] = 0;
  k.page_dtype = dtype;
  return keys_only(k);
}

Span means_span(const ako_paged_t& c, const float* means, const int64_t* st) {
  const int64_t st3[3] = {st[0], st[1], 0};
  return span_4d(means, c.num_pages, c.kv_heads, 1, c.head_dim, st3, 4);
}

int select_common(const char* fn, const ako_paged_t& cache, int64_t q_heads, int64_t count, int dtype,
                  ako::PagedSelectArgs* a, bool* empty) {
  if (const int rc = paged_common(fn, &cache, q_heads, dtype, &a->c, empty)) return rc;
  if (q_heads % cache.kv_heads)
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: %lld query heads are no multiple of %lld", fn, (long long)q_heads,
                (long long)cache.kv_heads);
  if (count < 1 || count > kMaxInt / 2) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: count must be 1 to 2^30", fn);
  // Of a launch's workgroups, 16 rows by 512 blocks each: work-items stay below 2^32.
  if (cache.table_width > (int64_t(1) << 28) / cache.kv_heads)
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: more than 2^28 blocks and key heads", fn);
  a->q_heads = q_heads;
  a->count = count;
  a->dtype = dtype;
  return AKO_OK;
}

}  // namespace
}  // extern "C++"

int ako_paged_means_fwd(const ako_paged_t* cache, float* means, const int64_t* means_strides, int dtype, void* stream) {
  const char* fn = "ako_paged_means_fwd";
  if (!cache) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: null cache", fn);
  const ako_paged_t c = keys_only(*cache);
  if (c.page_dtype == AKO_DTYPE_E4M3) dtype = AKO_DTYPE_F32;
  ako::PagedMeansArgs a{};
  bool empty = false;
  if (const int rc = paged_common(fn, &c, 0, dtype, &a.c, &empty)) return rc;
  if (empty || c.num_pages == 0) return AKO_OK;
  if (!means || !means_strides) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
  if (means_strides[0] < 0 || means_strides[1] < 0) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: negative stride", fn);
  const int64_t st3[3] = {means_strides[0], means_strides[1], 0};
  if (!distinct_rows(c.num_pages, c.kv_heads, 1, c.head_dim, st3))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: rows of the means overlap", fn);
  const Span m = means_span(c, means, means_strides);
  const PagedSpans held(&c, dtype);
  if (!m.ok || !held.ok) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: sizes and strides overflow the address space", fn);
  if (held.meets(m)) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: the means overlap another buffer", fn);
  a.means = means;
  a.ms[0] = means_strides[0];
  a.ms[1] = means_strides[1];
  a.dtype = dtype;
  return hip_status(ako::launch_paged_means(a, static_cast<hipStream_t>(stream)), fn);
}

int ako_paged_select_fwd(const ako_paged_t* cache, const void* q, const int64_t* q_strides, int64_t q_heads,
                         const float* means, const int64_t* means_strides, int32_t* blocks, int64_t count, int64_t first,
                         int64_t last, void* workspace, int64_t workspace_bytes, int dtype, void* stream) {
  const char* fn = "ako_paged_select_fwd";
  if (!cache) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: null cache", fn);
  ako::PagedSelectArgs a{};
  bool empty = false;
  const ako_paged_t c = no_pages(*cache, means, dtype);
  if (c.num_pages > 0 && c.tokens > 0 && !means) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: null means", fn);
  if (const int rc = select_common(fn, c, q_heads, count, dtype, &a, &empty)) return rc;
  if (first < 0 || last < 1 || first > count || last > count - first)
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: first must be >= 0, last >= 1 and count >= first + last", fn);
  if (empty) return AKO_OK;
  if ((q_heads > 0 && !q) || !q_strides || !blocks || !means_strides)
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
  if (q_strides[0] < 0 || q_strides[1] < 0 || q_strides[2] < 0 || means_strides[0] < 0 || means_strides[1] < 0)
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: negative stride", fn);
  const int64_t need = ako::paged_select_workspace(a);
  if (workspace_bytes < need || (need > 0 && (!workspace || !aligned(workspace, 16))))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: needs a 16-byte aligned workspace of %lld bytes, got %lld", fn,
                (long long)need, (long long)workspace_bytes);
  const int64_t per = c.cu_seqlens ? c.tokens : c.tokens / c.n_seqs;
  const __int128 out_bytes = static_cast<__int128>(c.tokens) * c.kv_heads * count * 4;
  const Span o = span_bytes(blocks, out_bytes), w = span_bytes(workspace, need);
  Span in[2];
  int n_in = 0;
  if (q_heads > 0)
    in[n_in++] = span_4d(q, c.cu_seqlens ? 1 : c.n_seqs, per, q_heads, c.head_dim, q_strides, ako::dtype_bytes(dtype));
  if (c.num_pages > 0) in[n_in++] = means_span(c, means, means_strides);
  const PagedSpans held(&c, dtype);
  bool ok = o.ok && w.ok && held.ok, apart = !overlap(o, w) && !held.meets_index(o) && !held.meets_index(w);
  for (int i = 0; i < n_in; ++i) {
    ok = ok && in[i].ok;
    apart = apart && !overlap(o, in[i]) && !overlap(w, in[i]);
  }
  if (!ok) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: sizes and strides overflow the address space", fn);
  if (!apart) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: blocks or the workspace overlap another buffer", fn);
  a.q = q;
  a.means = means;
  for (int i = 0; i < 3; ++i) a.qs[i] = q_strides[i];
  a.ms[0] = means_strides[0];
  a.ms[1] = means_strides[1];
  a.first = first;
  a.last = last;
  a.out = blocks;
  a.workspace = workspace;
  return hip_status(ako::launch_paged_select(a, static_cast<hipStream_t>(stream)), fn);
}

int64_t ako_paged_select_workspace(const ako_paged_t* cache, int64_t q_heads, int64_t count, int dtype) {
  const char* fn = "ako_paged_select_workspace";
  ako::PagedSelectArgs a{};
  bool empty = false;
  if (!cache) {
    fail(AKO_ERR_INVALID_ARGUMENT, "%s: null cache", fn);
    return -1;
  }
  const ako_paged_t c = no_pages(*cache, cache, dtype);
  if (select_common(fn, c, q_heads, count, dtype, &a, &empty)) return -1;
  return empty ? 0 : ako::paged_select_workspace(a);
}

// --------------------------------------------------------------- sampling --
static constexpr int64_t kMaxVocab = int64_t(1) << 22;

int64_t ako_sample_workspace(int64_t rows, int64_t vocab, int dtype) {
  if (!valid_dtype(dtype)) {
    fail(AKO_ERR_UNSUPPORTED, "ako_sample_workspace: unknown dtype code %d", dtype);
    return -1;
  }
  if (rows < 0 || rows > kMaxInt || vocab < 1 || vocab > kMaxVocab) {
    fail(AKO_ERR_INVALID_ARGUMENT, "ako_sample_workspace: rows must be 0 to 2^31-1 and vocab 1 to %lld", (long long)kMaxVocab);
    return -1;
  }
  return rows == 0 ? 0 : ako::sample_workspace(rows, vocab);
}

int ako_sample_fwd(const void* logits, const float* uniform, const float* temperature, float temperature_all,
                   const int32_t* top_k, int32_t top_k_all, const float* top_p, float top_p_all, const float* min_p,
                   float min_p_all, int64_t* out, int64_t rows, int64_t vocab, int64_t row_stride, void* workspace,
                   int64_t workspace_bytes, int dtype, void* stream) {
  const char* fn = "ako_sample_fwd";
  if (!valid_dtype(dtype)) return fail(AKO_ERR_UNSUPPORTED, "%s: unknown dtype code %d", fn, dtype);
  if (rows < 0 || rows > kMaxInt) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: rows must be 0 to 2^31-1", fn);
  if (vocab < 1 || vocab > kMaxVocab)
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: vocab must be 1 to %lld, got %lld", fn, (long long)kMaxVocab, (long long)vocab);
  if (!temperature && !(temperature_all >= 0.0f))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: temperature must be >= 0", fn);
  if (!top_k && top_k_all < 0) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: top_k must be >= 0", fn);
  if ((!top_p && !(top_p_all >= 0.0f && top_p_all <= 1.0f)) || (!min_p && !(min_p_all >= 0.0f && min_p_all <= 1.0f)))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: top_p and min_p must be 0 to 1", fn);
  if (rows == 0) return AKO_OK;
  if (!logits || !uniform || !out) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
  if (row_stride < 0) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: negative row stride", fn);
  const Span in = span_2d(logits, rows, vocab, row_stride, ako::dtype_bytes(dtype));
  const Span o = span_2d(out, 1, rows, rows, 8);
  const int64_t need = ako::sample_workspace(rows, vocab);
  if (workspace_bytes < need || (need > 0 && (!workspace || !aligned(workspace, 16))))
    return fail(AKO_ERR_INVALID_ARGUMENT, "%s: needs a 16-byte aligned workspace of %lld bytes, got %lld", fn,
                (long long)need, (long long)workspace_bytes);
  const Span ws = span_bytes(workspace, need);
  const void* const per_row[5] = {uniform, temperature, top_k, top_p, min_p};
  bool ok = in.ok && o.ok && ws.ok, apart = !overlap(o, in) && !overlap(ws, in) && !overlap(ws, o);
  for (const void* p : per_row) {
    if (!p) continue;
    const Span s = span_2d(p, 1, rows, rows, 4);
    ok = ok && s.ok;
    apart = apart && !overlap(o, s) && !overlap(ws, s);
  }
  if (!ok) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: sizes and strides overflow the address space", fn);
  if (!apart) return fail(AKO_ERR_INVALID_ARGUMENT, "%s: out or the workspace overlaps another buffer", fn);
  ako::SampleArgs a{};
  a.x = logits;
  a.rows = rows;
  a.vocab = vocab;
  a.stride = row_stride;
  a.u = uniform;
  a.temperatures = temperature;
  a.top_ks = top_k;
  a.top_ps = top_p;
  a.min_ps = min_p;
  a.temperature = temperature_all;
  a.top_k = top_k_all;
  a.top_p = top_p_all;
  a.min_p = min_p_all;
  a.out = out;
  a.workspace = workspace;
  a.dtype = dtype;
  return hip_status(ako::launch_sample(a, static_cast<hipStream_t>(stream)), fn);
}

}  // extern "C"

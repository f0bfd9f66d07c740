/*
 * ako_hip.h - C ABI of the MI355X (gfx950) AKO candidate kernels.
 *
 * One shared library, libako_hip.so, exports the entry points below. They
 * take plain device pointers, element counts and strides, a dtype code and a
 * hipStream_t passed as void*. No PyTorch (or any C++) type crosses this
 * boundary, so the library can be bound from ctypes, cgo or JNI alike.
 *
 * Each entry point replaces one Triton candidate of the reference
 * (Farx1/AKO); the citation next to each declaration names the host wrapper
 * and kernel whose contract it takes over.
 *
 * Conventions shared by every entry point
 *   - Pointers are device pointers (hipMalloc'd or from a caching allocator).
 *   - Strides are in ELEMENTS, not bytes. The innermost dimension (hidden,
 *     head_dim, n) must be contiguous.
 *   - Outputs must not overlap any input; overlapping ranges are rejected.
 *   - Work is enqueued on `stream` (NULL = the default stream) and the call
 *     returns without synchronising. Launch errors are reported; errors that
 *     happen later on the device surface at the caller's next sync.
 *   - Arithmetic is fp32 internally for every storage dtype; results are
 *     rounded to the output dtype with round-to-nearest-even.
 *   - Return value: AKO_OK (0) or a nonzero ako_status_t; ako_last_error()
 *     then returns a message (thread-local, valid until the next call on the
 *     same thread).
 *   - Empty work (rows == 0, hidden == 0, ...) returns AKO_OK and launches
 *     nothing.
 */
#ifndef AKO_HIP_H
#define AKO_HIP_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define AKO_ABI_VERSION 1

typedef enum {
  AKO_DTYPE_F32 = 0,
  AKO_DTYPE_F16 = 1,
  AKO_DTYPE_BF16 = 2,
  AKO_DTYPE_E4M3 = 3 /* pages of a paged cache only: OCP e4m3 with scale codes */
} ako_dtype_t;

typedef enum {
  AKO_OK = 0,
  AKO_ERR_INVALID_ARGUMENT = 1, /* null pointer, negative size, bad stride, overlap */
  AKO_ERR_UNSUPPORTED = 2,      /* dtype combination or style not provided      */
  AKO_ERR_HIP = 3,              /* the HIP runtime reported an error            */
  AKO_ERR_NO_DEVICE = 4         /* no usable GPU in this process                 */
} ako_status_t;

typedef enum {
  AKO_ROPE_NEOX = 0,        /* pairs (i, i + head_dim/2) */
  AKO_ROPE_INTERLEAVED = 1  /* pairs (2i, 2i + 1)        */
} ako_rope_style_t;

/* Library identity: AKO_ABI_VERSION, and the HIP runtime version
 * (hipRuntimeGetVersion) of the runtime this library is bound to. */
int ako_abi_version(void);
int ako_hip_runtime_version(void);
const char* ako_build_info(void);
const char* ako_last_error(void);

/*
 * Identity of GPU `device` for the selection cache key, written into buf as
 * one NUL-terminated line of key=value fields separated by ';':
 *   name=<hipDeviceProp_t.name>;arch=<gcnArchName>;cus=<CUs>;
 *   clock_khz=<peak engine clock>;mem_bytes=<HBM bytes>;hip_driver=<hipDriverGetVersion>
 * Replaces the device-name probe of ako/dispatcher/hardware.py:134-193 (CUDA
 * runtime attributes and nvidia-smi). The marketing name that HIP reports can
 * be a generic "AMD Radeon Graphics" for every part, so callers key by the
 * other fields too. Returns AKO_ERR_INVALID_ARGUMENT when buf is too small.
 */
int ako_device_identity(int device, char* buf, int64_t buf_len);

/*
 * RMSNorm over the last dimension:
 *   y[r, :] = to_dtype( (x[r, :] * rsqrt(sum(x[r, :]^2) / hidden + eps)) * w[:] )
 * x, y: dtype; w: w_dtype (== dtype, or AKO_DTYPE_F32).
 * Replaces rmsnorm_triton + _rmsnorm_kernel_impl
 * (ako/ops/rmsnorm_triton.py:56-81, 139-157). Unlike the reference there is
 * no hidden-size limit (the reference raised above 65536,
 * ako/ops/rmsnorm_triton.py:28,130-133).
 */
int ako_rmsnorm_fwd(const void* x, const void* w, void* y,
                    int64_t rows, int64_t hidden,
                    int64_t x_row_stride, int64_t y_row_stride,
                    float eps, int dtype, int w_dtype, void* stream);

/*
 * Residual-add + RMSNorm:
 *   s = to_dtype(x + residual)       (the sum is rounded to the storage dtype)
 *   residual_out = s
 *   y = RMSNorm(s, w, eps)
 * Replaces rmsnorm_residual_triton + _rmsnorm_residual_kernel_impl
 * (ako/ops/rmsnorm_triton.py:83-117, 160-192) and matches the unfused
 * reference ako/ops/rmsnorm_ref.py:26-50.
 */
int ako_rmsnorm_residual_fwd(const void* x, const void* residual, const void* w,
                             void* y, void* residual_out,
                             int64_t rows, int64_t hidden,
                             int64_t x_row_stride, int64_t r_row_stride,
                             int64_t y_row_stride, int64_t rout_row_stride,
                             float eps, int dtype, int w_dtype, void* stream);

/*
 * RMSNorm of a row whose hidden dimension is split over tensor-parallel
 * ranks: the per-rank halves of a fused all-reduce + residual + RMSNorm. The
 * reference has no tensor parallelism, so neither has a counterpart there;
 * together they compute rmsnorm_residual_ref / rmsnorm_ref
 * (ako/ops/rmsnorm_ref.py:8-50) on the whole row, up to the order of the
 * fp32 sum of squares:
 *   partial:  s = x (+ residual, rounded to dtype, written to residual_out;
 *             both NULL for plain RMSNorm), partial_ss[row] = sum of s^2 over
 *             the rank's `shard` elements (fp32);
 *   (the caller sums partial_ss over the ranks, e.g. one all-reduce)
 *   apply:    y = to_dtype((s * rsqrt(total_ss[row] * (1/hidden) + eps)) * w)
 *             on the rank's slice, with `hidden` the full row length.
 * Row strides in elements; partial_ss / total_ss hold `rows` floats.
 */
int ako_rmsnorm_shard_partial_fwd(const void* x, const void* residual, void* residual_out,
                                  float* partial_ss, int64_t rows, int64_t shard,
                                  int64_t x_row_stride, int64_t r_row_stride,
                                  int64_t rout_row_stride, int dtype, void* stream);
int ako_rmsnorm_shard_apply_fwd(const void* s, const void* w, const float* total_ss, void* y,
                                int64_t rows, int64_t shard, int64_t hidden,
                                int64_t s_row_stride, int64_t y_row_stride, float eps,
                                int dtype, int w_dtype, void* stream);

/*
 * Rotary position embedding of x[batch, seq, heads, head_dim]:
 *   for each pair (a, b) of a head at position s, with c = cos[s, i],
 *   n = sin[s, i]:   a' = a*c - b*n,   b' = a*n + b*c     (fp32)
 * cos/sin: [seq, head_dim/2] rows `table_row_stride` apart, dtype
 * `table_dtype` (F32, F16 or BF16, independent of x's dtype).
 * x strides (batch, seq, head) and y strides likewise, in elements.
 * Replaces rope_triton + _rope_kernel_impl (ako/ops/rope_triton.py:32-80,
 * 97-156); semantics of ako/ops/rope_ref.py:73-107.
 */
int ako_rope_fwd(const void* x, const void* cos_table, const void* sin_table, void* y,
                 int64_t batch, int64_t seq, int64_t heads, int64_t head_dim,
                 int64_t x_stride_b, int64_t x_stride_s, int64_t x_stride_h,
                 int64_t y_stride_b, int64_t y_stride_s, int64_t y_stride_h,
                 int64_t table_row_stride,
                 int dtype, int table_dtype, int style, void* stream);

/*
 * RoPE of a query/key pair sharing the tables, in ONE launch (the reference
 * runs two, ako/ops/rope.py:45-58). q is [batch, seq, q_heads, head_dim],
 * k is [batch, seq, k_heads, head_dim]; strides as in ako_rope_fwd.
 */
int ako_rope_qk_fwd(const void* q, const void* k, const void* cos_table, const void* sin_table,
                    void* q_out, void* k_out,
                    int64_t batch, int64_t seq, int64_t q_heads, int64_t k_heads,
                    int64_t head_dim,
                    const int64_t* q_strides, const int64_t* k_strides,
                    const int64_t* q_out_strides, const int64_t* k_out_strides,
                    int64_t table_row_stride,
                    int dtype, int table_dtype, int style, void* stream);

/*
 * RoPE of a query/key pair with the rotated keys (and the values, copied)
 * written straight into a KV cache, in ONE launch. This is the fused consumer
 * the reference's decoder performs as rope(q), rope(k) and a cache append
 * (ako/models/decoder.py:173-177, KVCache.update at :84-93).
 *   position of token s:  p = *pos + s   (pos: one int64 in device memory,
 *                                         read by the kernel, so a captured
 *                                         launch follows a moving position)
 *   q_out[b, s, h]      = rope(q[b, s, h], row p of cos/sin)
 *   k_cache[b, h, slot p] = rope(k[b, s, h], row p)
 *   v_cache[b, h, slot p] = v[b, s, h]          (v and v_cache may both be NULL)
 * q/k/v/q_out strides are (batch, seq, head); cache_strides (batch, slot,
 * head) are shared by both caches, in elements. The tables hold table_rows
 * >= cache_len rows. A token whose p falls outside [0, cache_len) writes no
 * cache slot, and its q_out rows are filled with NaN; keeping
 * *pos + seq <= cache_len is the caller's contract (the reference's unfused
 * composition raises an index error there, which a position held in device
 * memory cannot do).
 */
int ako_rope_qk_cache_fwd(const void* q, const void* k, const void* v,
                          const void* cos_table, const void* sin_table,
                          void* q_out, void* k_cache, void* v_cache, const int64_t* pos,
                          int64_t batch, int64_t seq, int64_t q_heads, int64_t kv_heads,
                          int64_t head_dim,
                          const int64_t* q_strides, const int64_t* k_strides,
                          const int64_t* v_strides, const int64_t* q_out_strides,
                          const int64_t* cache_strides,
                          int64_t cache_len, int64_t table_rows, int64_t table_row_stride,
                          int dtype, int table_dtype, int style, void* stream);

/*
 * RMSNorm of every head of q and k with a weight per element, and RoPE, in one
 * pass: for each head x of q (w = q_weight) and of k (w = k_weight)
 *   y = (x * rsqrt(sum(x^2) / head_dim + eps)) * w      (fp32)
 * and y's pairs rotated as by ako_rope_fwd, the result rounded once. The
 * reference has no such pass; it is rmsnorm_ref (ako/ops/rmsnorm_ref.py:8-24) over
 * heads, then rope_ref (ako/ops/rope_ref.py:73-107), without the rounding between.
 * q and k are [batch, seq, heads, head_dim] with strides as in ako_rope_fwd (either
 * may have no heads), the outputs dense. head_dim is even, at most 512. The weights
 * are of dtype or AKO_DTYPE_F32.
 */
int ako_rmsnorm_rope_qk_fwd(const void* q, const void* k, const void* q_weight, const void* k_weight,
                            const void* cos_table, const void* sin_table, void* q_out, void* k_out,
                            int64_t batch, int64_t seq, int64_t q_heads, int64_t k_heads,
                            int64_t head_dim, const int64_t* q_strides, const int64_t* k_strides,
                            int64_t table_row_stride, float eps, int dtype, int w_dtype,
                            int table_dtype, int style, void* stream);

/*
 * SwiGLU activation: y = to_dtype( silu(gate) * up ), silu(g) = g / (1 + e^-g),
 * over [rows, n] with row strides in elements.
 * Replaces swiglu_triton + _swiglu_kernel_impl
 * (ako/ops/swiglu_triton.py:27-81); semantics of ako/ops/swiglu_ref.py:16-32.
 * No width limit (the reference raised above 65536).
 */
int ako_swiglu_fwd(const void* gate, const void* up, void* y,
                   int64_t rows, int64_t n,
                   int64_t gate_row_stride, int64_t up_row_stride, int64_t y_row_stride,
                   int dtype, void* stream);

/*
 * A paged key/value cache and the token rows of one step. The reference has
 * no counterpart (its decoder re-concatenates dense caches,
 * ako/models/decoder.py:84-93); the step's semantics are those of
 * ako/models/decoder.py:173-185 with the caches in pages.
 *
 * Keys and values lie in pools of pages, [num_pages, kv_heads, page_size,
 * head_dim] in any strides with head_dim contiguous. Position p of sequence i
 * is slot p % page_size of page block_table[i][p / page_size]; an entry
 * outside [0, num_pages) is a page that is not there. seq_lens[i] counts the
 * positions of sequence i with this step's tokens. A step has `tokens` rows:
 * with cu_seqlens, rows cu_seqlens[i] .. cu_seqlens[i+1]-1 are the last
 * positions of sequence i (cu_seqlens[0] = 0, ascending; rows from
 * cu_seqlens[n_seqs] on are padding); without, sequence i has the rows
 * i*(tokens/n_seqs) .. (i+1)*(tokens/n_seqs)-1. A row whose position would be
 * negative (a sequence shorter than its rows) is padding too. block_table,
 * seq_lens and cu_seqlens are read on the device, so that a captured step can
 * be replayed as they change; whatever they hold, no kernel reads or writes
 * outside the tensors.
 *
 * page_dtype is the rows' own dtype, or AKO_DTYPE_E4M3: one byte per element
 * and, for each 32 elements of a row, an E8M0 scale code c (2^(c-127); 255 is NaN) in
 * k_scales / v_scales [num_pages, kv_heads, page_size, ceil(head_dim/32)],
 * last dimension contiguous. A block is written with the smallest code >= 1
 * under which none of its finite elements passes 448, elements rounded to
 * nearest even; infinities and NaN are written as NaN.
 *
 * head_dim is a multiple of 16 up to 256. Stride triples are page, head, slot.
 */
typedef struct {
  void* k_pages;
  void* v_pages;
  void* k_scales;            /* NULL unless page_dtype is AKO_DTYPE_E4M3 */
  void* v_scales;
  const int32_t* block_table; /* [n_seqs, table_width], rows table_stride apart */
  const int32_t* seq_lens;    /* [n_seqs] */
  const int32_t* cu_seqlens;  /* [n_seqs + 1], or NULL */
  int64_t k_strides[3], v_strides[3];
  int64_t k_scale_strides[3], v_scale_strides[3];
  int64_t num_pages, kv_heads, page_size, head_dim;
  int64_t n_seqs, table_width, table_stride;
  int64_t tokens;
  int32_t page_dtype;
} ako_paged_t;

/*
 * RoPE of the step's q and k at their positions: rotated q to q_out
 * ([tokens, q_heads, head_dim], dense), rotated k and unrotated v to their
 * slots. k and v have cache->kv_heads heads. Stride triples of q, k and v are
 * sequence, token, head; with cu_seqlens the first is not used. The tables
 * hold positions 0 .. table_rows-1. The rows of q_out of padding are zero; a
 * row whose page is not there, or whose position the block table or the
 * tables do not cover, is written to no slot and its row of q_out is NaN. Rows
 * of one step must not share a slot.
 */
int ako_rope_qk_paged_fwd(const void* q, const void* k, const void* v,
                          const void* cos_table, const void* sin_table, void* q_out,
                          const ako_paged_t* cache, int64_t q_heads,
                          const int64_t* q_strides, const int64_t* k_strides,
                          const int64_t* v_strides, int64_t table_rows, int64_t table_row_stride,
                          int dtype, int table_dtype, int style, void* stream);

/*
 * The same with every head of q and k through its RMSNorm first, as in
 * ako_rmsnorm_rope_qk_fwd: nothing is rounded between the norm and the rotation, nor
 * between those and an e4m3 page. Values are stored as they are.
 */
int ako_rmsnorm_rope_qk_paged_fwd(const void* q, const void* k, const void* v,
                                  const void* q_weight, const void* k_weight,
                                  const void* cos_table, const void* sin_table, void* q_out,
                                  const ako_paged_t* cache, int64_t q_heads,
                                  const int64_t* q_strides, const int64_t* k_strides,
                                  const int64_t* v_strides, int64_t table_rows,
                                  int64_t table_row_stride, float eps, int dtype, int w_dtype,
                                  int table_dtype, int style, void* stream);

/*
 * The keys and values stored at the rows' positions, as dense [tokens,
 * kv_heads, head_dim] tensors of dtype (which must be page_dtype unless that
 * is AKO_DTYPE_E4M3). Rows that are padding or have no page are zero.
 */
int ako_paged_read_fwd(const ako_paged_t* cache, void* k_out, void* v_out, int dtype, void* stream);

/*
 * Attention of the step's rows over what their sequences hold. Head h of q
 * attends to head h / (q_heads / kv_heads) of the cache; a row at position p
 * sees the positions j <= p with (window == 0, or j > p - window, or
 * j < sinks), except those whose page is not there:
 *   out = to_dtype( sum_j softmax_j(scale * q.k_j) v_j ),
 * zero where a row sees nothing (padding), NaN where all it sees scores
 * -infinity. Positions a row does not see have no influence on it, whatever
 * they and their scale codes hold. An infinity or NaN among the values that a
 * row sees makes the row's element of it that infinity or NaN (an infinity
 * whose weight vanishes may give NaN). out is [tokens, q_heads, head_dim],
 * dense; q's strides are sequence, token, head. e4m3 pages are read as values
 * of dtype. workspace holds ako_paged_attention_workspace bytes of device
 * memory, 16-byte aligned, that nothing else uses until the work on `stream`
 * is done.
 */
int ako_paged_attention_fwd(const void* q, const int64_t* q_strides, void* out,
                            const ako_paged_t* cache, int64_t q_heads, float scale,
                            int64_t window, int64_t sinks, void* workspace,
                            int64_t workspace_bytes, int dtype, void* stream);

/* Bytes of workspace for such a call (0: none); -1 for arguments it refuses. */
int64_t ako_paged_attention_workspace(const ako_paged_t* cache, int64_t q_heads, int dtype);

/*
 * The same over listed blocks only: a row at position p of key head `head` sees the
 * positions j <= p whose block j / page_size is among blocks[row][head][0 .. count-1], int32,
 * dense (as ako_paged_select_fwd writes it). The list is a set: in any order, and a block that
 * stands there twice counts once; numbers below 0 or past the table name nothing. A row with
 * no such position is zero.
 */
int ako_paged_attention_blocks_fwd(const void* q, const int64_t* q_strides, void* out,
                                   const ako_paged_t* cache, int64_t q_heads, float scale,
                                   const int32_t* blocks, int64_t count, void* workspace,
                                   int64_t workspace_bytes, int dtype, void* stream);

/* Bytes of workspace for such a call (0: none); -1 for arguments it refuses. */
int64_t ako_paged_attention_blocks_workspace(const ako_paged_t* cache, int64_t q_heads,
                                             int64_t count, int dtype);

/*
 * The mean of the keys of every page that the step's rows fill: for a row at the last
 * slot of its page, means[page][head] = sum over the page's slots of the keys as stored / page_size
 * (fp32; e4m3 keys times their scales). means is [num_pages, kv_heads, head_dim] floats,
 * means_strides those of page and head; no other page's means are touched. The cache's
 * v_pages, v_scales and their strides are not used; the pages are of dtype, or e4m3
 * (dtype is then not used).
 */
int ako_paged_means_fwd(const ako_paged_t* cache, float* means, const int64_t* means_strides,
                        int dtype, void* stream);

/*
 * For each row and key head the blocks (pages) to attend to, into
 * blocks[row][head][0 .. count-1], ascending, -1 behind the last. A row at position p may take
 * the blocks 0 .. p / page_size whose page is there; all of them, if they are no more
 * than count, else count of them: the first `first`, the last `last` up to its own,
 * and of the others those with the largest scores
 *   sum over the heads h that read key head `head` of q[row][h] . means[page][head],
 * of equal ones the lowest blocks (64-bit sums, in an order that hangs on how many rows a
 * sequence has: scores closer than some 2^-50 of the size of their terms may change places with it; NaN counts as
 * -infinity). first >= 0,
 * last >= 1, count >= first + last. Rows that are padding get -1 only. Of the cache, the pages, scales and their
 * strides are not used and page_dtype is dtype, that of q. workspace
 * holds ako_paged_select_workspace bytes, 16-byte aligned, that nothing else uses until the
 * work on `stream` is done.
 */
int ako_paged_select_fwd(const ako_paged_t* cache, const void* q, const int64_t* q_strides,
                         int64_t q_heads, const float* means, const int64_t* means_strides,
                         int32_t* blocks, int64_t count, int64_t first, int64_t last,
                         void* workspace, int64_t workspace_bytes, int dtype, void* stream);

/* Bytes of workspace for such a call (0: none); -1 for arguments it refuses. */
int64_t ako_paged_select_workspace(const ako_paged_t* cache, int64_t q_heads, int64_t count,
                                   int dtype);

/*
 * A token for each of `rows` rows of `vocab` logits (1 to 2^22), from one uniform number each.
 * With w_i = e^((x_i - max x) / temperature), in descending order of the logits (of
 * equal ones the lowest index first) the first top_k tokens stay (0 or less: all), of
 * those the shortest run from the front that weighs at least top_p of them all
 * (1 or more: all; at least one), and of those the ones with w_i >= min_p (0 or less: all). out is
 * the first token, by index, at which the sum of the weights of what stays, so far, passes
 * uniform times their whole sum; for numbers from 1 on the last that weighs anything.
 * temperature 0 or less, or NaN, takes the largest logit's first token. Tokens of -infinity
 * or NaN are never drawn; where there are no others out is -1. Among several +infinities only
 * those are drawn, alike. Weights are sums of whole numbers, 2^-46 of the largest at 131072
 * tokens and finer below: the token does not depend on how the work was divided.
 * temperature, top_k, top_p and min_p hold one value for each row, or are NULL and the
 * value behind them holds for all rows (temperature_all >= 0 and not NaN, the others' in
 * [0, 1], top_k_all >= 0). row_stride: elements between rows. workspace holds
 * ako_sample_workspace bytes, 16-byte aligned, that nothing else uses until the work on `stream` is done. The reference has no
 * counterpart (its decoder returns hidden states, ako/models/decoder.py:261-266).
 */
int ako_sample_fwd(const void* logits, const float* uniform, const float* temperature,
                   float temperature_all, const int32_t* top_k, int32_t top_k_all,
                   const float* top_p, float top_p_all, const float* min_p, float min_p_all,
                   int64_t* out, int64_t rows, int64_t vocab, int64_t row_stride,
                   void* workspace, int64_t workspace_bytes, int dtype, void* stream);

/* Bytes of workspace for such a call (0: none); -1 for sizes it refuses. */
int64_t ako_sample_workspace(int64_t rows, int64_t vocab, int dtype);

/*
 * Launch-shape override for tuning sweeps and tests (no counterpart in the
 * reference, whose Triton autotuner explored num_warps itself); production
 * callers leave it alone. op: 0 = rmsnorm and rmsnorm_residual, 1 = rope,
 * 2 = swiglu, 3 = paged attention. key/value pairs are documented in the kernel sources; value 0
 * restores the built-in heuristic. Process-wide. Each key is an atomic int,
 * so the call is safe from any host thread: a launch that runs concurrently
 * sees each key's value from before or after the call (a launch concurrent
 * with several calls may mix their values).
 */
int ako_set_tuning(int op, int key, int value);

/*
 * Timing hook for benchmarks (no counterpart in the reference, which timed
 * through Triton's do_bench): arms two HIP events for the next kernel launch
 * that the calling host thread makes through any entry point above. That
 * launch goes out through hipExtLaunchKernelGGL with the pair, which binds
 * both events to the dispatch itself: hipEventElapsedTime(start, stop) is
 * then the kernel's own start-to-end time, the figure a kernel trace reports,
 * without the marker packets that an hipEventRecord on each side would queue
 * around it. The events are the caller's (hipEventCreate, timing enabled);
 * an entry point that makes several launches (inputs past 2^31 work-items,
 * attention that joins split key ranges) times its first. Arming replaces a pair that no launch has taken. Do
 * not arm a pair while the thread captures a stream into a graph: the next
 * launch takes it whether or not it is captured.
 * start and stop both NULL disarms: the return value is then 1 when a pair
 * was still armed (no launch took it), else AKO_OK. Exactly one NULL is
 * AKO_ERR_INVALID_ARGUMENT.
 */
int ako_time_next_launch(void* start_event, void* stop_event);

#ifdef __cplusplus
}
#endif

#endif /* AKO_HIP_H */

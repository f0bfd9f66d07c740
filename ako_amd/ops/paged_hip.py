"""HIP path of the paged-cache operations (gfx950 kernels).

Each function has the host work once in C++ (``_ako_torch``) and once here,
through ctypes, with the same checks and messages. Outputs are fresh; the
attention's workspace comes from torch's allocator on the launching stream, so
that calls on different streams, and captured graphs, never share one.
"""

from __future__ import annotations

import ctypes

import torch

from ako_amd import _native
from ako_amd.ops import paged_ref as ref
from ako_amd.ops._hip_common import DT, call, gpu_index, lib, raw_stream
from ako_amd.ops.qk_norm import kernel_weights
from ako_amd.ops.rope_hip import _head_view, _table, _table_stride

_I64x3 = ctypes.c_int64 * 3


def _cache(k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, cu_seqlens, tokens: int):
    num_pages, kv_heads, page_size, head_dim = k_pages.shape
    none = _I64x3()
    st = lambda t: none if t is None else _I64x3(*t.stride()[:3])  # noqa: E731
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    return _native.PagedCache(
        k_pages.data_ptr(), v_pages.data_ptr(), ptr(k_scales), ptr(v_scales), block_table.data_ptr(),
        seq_lens.data_ptr(), ptr(cu_seqlens), st(k_pages), st(v_pages), st(k_scales), st(v_scales),
        num_pages, kv_heads, page_size, head_dim, block_table.shape[0], block_table.shape[1],
        block_table.stride(0) if block_table.shape[0] > 1 else block_table.shape[1], tokens,
        DT.get(k_pages.dtype, _native.E4M3_CODE))


def _row_strides(x: torch.Tensor) -> ctypes.Array:
    return _I64x3(*(x.stride()[:3] if x.dim() == 4 else (0, x.stride(0), x.stride(1))))


def _tokens(x: torch.Tensor) -> int:
    return x.shape[0] * x.shape[1] if x.dim() == 4 else x.shape[0]


def rope_qk_paged_hip(q, k, v, cos, sin, k_pages, v_pages, block_table, seq_lens, style="neox",
                      k_scales=None, v_scales=None, cu_seqlens=None, q_weight=None, k_weight=None, eps=1e-6) -> torch.Tensor:
    """Rotated (with weights, normed and rotated) q out, k and v into their pages, in one launch."""
    fast = _native.torch_binding()
    run = rope_qk_paged_hip_ctypes if fast is None else fast.rope_qk_paged
    return run(q, k, v, cos, sin, k_pages, v_pages, block_table, seq_lens, style, k_scales, v_scales, cu_seqlens,
               q_weight, k_weight, eps)


def rope_qk_paged_hip_ctypes(q, k, v, cos, sin, k_pages, v_pages, block_table, seq_lens, style="neox",
                             k_scales=None, v_scales=None, cu_seqlens=None, q_weight=None, k_weight=None,
                             eps=1e-6) -> torch.Tensor:
    fn = "rope_qk_paged_hip"
    index = gpu_index(q, fn)
    ref.refuse(fn, ref.cache_error(k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, cu_seqlens)
               or ref.write_error(q, k, v, cos, sin, k_pages, block_table, style, cu_seqlens)
               or ref.norm_error(q_weight, k_weight, eps, k_pages))
    qv, kv, vv = _head_view(q), _head_view(k), _head_view(v)
    c, s, st = _table_stride(_table(cos, index), _table(sin, index))
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    cache = _cache(k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, cu_seqlens, _tokens(q))
    step = (c.data_ptr(), s.data_ptr(), out.data_ptr(), ctypes.addressof(cache), q.shape[-2], _row_strides(qv),
            _row_strides(kv), _row_strides(vv), c.shape[0], st)
    types = (DT[c.dtype], _native.ROPE_STYLE_CODES[style], raw_stream(index))
    rows = (qv.data_ptr(), kv.data_ptr(), vv.data_ptr())
    if q_weight is None:
        status = call(index, lib().ako_rope_qk_paged_fwd, *rows, *step, DT[q.dtype], *types)
    else:
        qw, kw = kernel_weights(q_weight, k_weight, q.dtype)
        status = call(index, lib().ako_rmsnorm_rope_qk_paged_fwd, *rows, qw.data_ptr(), kw.data_ptr(), *step, eps,
                      DT[q.dtype], DT[qw.dtype], *types)
    if status:
        _native.check(status, fn)
    return out


def paged_read_hip(k_pages, v_pages, block_table, seq_lens, rows, dtype=None, k_scales=None, v_scales=None,
                   cu_seqlens=None) -> tuple[torch.Tensor, torch.Tensor]:
    """Dense keys and values of each sequence's last positions, in one launch."""
    fast = _native.torch_binding()
    if fast is not None:
        return fast.paged_read(k_pages, v_pages, block_table, seq_lens, rows, dtype, k_scales, v_scales, cu_seqlens)
    return paged_read_hip_ctypes(k_pages, v_pages, block_table, seq_lens, rows, dtype, k_scales, v_scales, cu_seqlens)


def paged_read_hip_ctypes(k_pages, v_pages, block_table, seq_lens, rows, dtype=None, k_scales=None, v_scales=None,
                          cu_seqlens=None) -> tuple[torch.Tensor, torch.Tensor]:
    fn = "paged_read_hip"
    index = gpu_index(k_pages, fn)
    ref.refuse(fn, ref.cache_error(k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, cu_seqlens)
               or ref.read_error(k_pages, rows, dtype))
    dtype = k_pages.dtype if dtype is None else dtype
    n, (_, kv_heads, _, head_dim) = block_table.shape[0], k_pages.shape
    lead = (rows,) if cu_seqlens is not None else (n, rows)
    k, v = (torch.empty(*lead, kv_heads, head_dim, dtype=dtype, device=k_pages.device) for _ in range(2))
    cache = _cache(k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, cu_seqlens, _tokens(k))
    status = call(index, lib().ako_paged_read_fwd, ctypes.addressof(cache), k.data_ptr(), v.data_ptr(), DT[dtype],
                  raw_stream(index))
    if status:
        _native.check(status, fn)
    return k, v


def paged_means_hip(k_pages, k_means, block_table, seq_lens, rows, k_scales=None, cu_seqlens=None) -> torch.Tensor:
    """Means of the pages that the step's rows fill, in one launch."""
    fast = _native.torch_binding()
    run = paged_means_hip_ctypes if fast is None else fast.paged_means
    return run(k_pages, k_means, block_table, seq_lens, rows, k_scales, cu_seqlens)


def paged_means_hip_ctypes(k_pages, k_means, block_table, seq_lens, rows, k_scales=None, cu_seqlens=None) -> torch.Tensor:
    fn = "paged_means_hip"
    index = gpu_index(k_pages, fn)
    ref.refuse(fn, ref.cache_error(k_pages, k_pages, k_scales, k_scales, block_table, seq_lens, cu_seqlens)
               or ref.means_error(k_means, k_pages) or ref.count_error(rows))
    tokens = rows if cu_seqlens is not None else block_table.shape[0] * rows
    cache = _cache(k_pages, k_pages, k_scales, k_scales, block_table, seq_lens, cu_seqlens, tokens)
    status = call(index, lib().ako_paged_means_fwd, ctypes.addressof(cache), k_means.data_ptr(),
                  _I64x3(*k_means.stride()[:2], 0), DT.get(k_pages.dtype, 0), raw_stream(index))
    if status:
        _native.check(status, fn)
    return k_means


def paged_select_hip(q, k_means, block_table, seq_lens, page_size, count, first=1, last=1, cu_seqlens=None) -> torch.Tensor:
    """The blocks that each row and key head attends to."""
    fast = _native.torch_binding()
    run = paged_select_hip_ctypes if fast is None else fast.paged_select
    return run(q, k_means, block_table, seq_lens, page_size, count, first, last, cu_seqlens)


def paged_select_hip_ctypes(q, k_means, block_table, seq_lens, page_size, count, first=1, last=1, cu_seqlens=None) -> torch.Tensor:
    fn = "paged_select_hip"
    index = gpu_index(q, fn)
    ref.refuse(fn, ref.select_error(q, k_means, block_table, seq_lens, page_size, count, first, last, cu_seqlens))
    qv = _head_view(q)
    out = torch.empty(*q.shape[:-2], k_means.shape[1], count, dtype=torch.int32, device=q.device)
    pages = ref.blocks_as_pages(k_means, page_size)
    cache = _cache(pages, pages, None, None, block_table, seq_lens, cu_seqlens, _tokens(q))
    cache.page_dtype = DT[q.dtype]
    at, heads, dt = ctypes.addressof(cache), q.shape[-2], DT[q.dtype]
    need = lib().ako_paged_select_workspace(at, heads, count, dt)
    space = torch.empty(need, dtype=torch.uint8, device=q.device) if need > 0 else None
    status = call(index, lib().ako_paged_select_fwd, at, qv.data_ptr(), _row_strides(qv), heads, k_means.data_ptr(),
                  _I64x3(*k_means.stride()[:2], 0), out.data_ptr(), count, first, last,
                  space.data_ptr() if space is not None else None, max(need, 0), dt, raw_stream(index))
    if status:
        _native.check(status, fn)
    return out


def paged_attention_hip(q, k_pages, v_pages, block_table, seq_lens, scale=None, window=None, sinks=0,
                        k_scales=None, v_scales=None, cu_seqlens=None, blocks=None) -> torch.Tensor:
    """Attention of a step's rows over their sequences' pages, or the listed ones of them."""
    fast = _native.torch_binding()
    run = paged_attention_hip_ctypes if fast is None else fast.paged_attention
    return run(q, k_pages, v_pages, block_table, seq_lens, scale, window, sinks, k_scales, v_scales, cu_seqlens, blocks)


def paged_attention_hip_ctypes(q, k_pages, v_pages, block_table, seq_lens, scale=None, window=None, sinks=0,
                               k_scales=None, v_scales=None, cu_seqlens=None, blocks=None) -> torch.Tensor:
    fn = "paged_attention_hip"
    index = gpu_index(q, fn)
    ref.refuse(fn, ref.cache_error(k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, cu_seqlens)
               or ref.rows_error("q", q, -1, k_pages, block_table, cu_seqlens))
    scale = k_pages.shape[3] ** -0.5 if scale is None else scale
    ref.refuse(fn, ref.attention_error(q, k_pages, scale, window, sinks)
               or ref.blocks_error(q, k_pages, blocks, window, sinks))
    qv = _head_view(q)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    cache = _cache(k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, cu_seqlens, _tokens(q))
    at, heads, dt = ctypes.addressof(cache), q.shape[-2], DT[q.dtype]
    if blocks is None:
        need = lib().ako_paged_attention_workspace(at, heads, dt)
    else:
        blocks = blocks.contiguous()
        need = lib().ako_paged_attention_blocks_workspace(at, heads, blocks.shape[-1], dt)
    space = torch.empty(need, dtype=torch.uint8, device=q.device) if need > 0 else None
    work = (space.data_ptr() if space is not None else None, max(need, 0), dt, raw_stream(index))
    step = (qv.data_ptr(), _row_strides(qv), out.data_ptr(), at, heads, scale)
    if blocks is None:
        status = call(index, lib().ako_paged_attention_fwd, *step, window or 0, sinks, *work)
    else:
        status = call(index, lib().ako_paged_attention_blocks_fwd, *step, blocks.data_ptr(), blocks.shape[-1], *work)
    if status:
        _native.check(status, fn)
    return out

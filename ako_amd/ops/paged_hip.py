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
                      k_scales=None, v_scales=None, cu_seqlens=None) -> torch.Tensor:
    """Rotated q out, rotated k and v into their pages, in one launch."""
    fast = _native.torch_binding()
    if fast is not None:
        return fast.rope_qk_paged(q, k, v, cos, sin, k_pages, v_pages, block_table, seq_lens, style,
                                  k_scales, v_scales, cu_seqlens)
    return rope_qk_paged_hip_ctypes(q, k, v, cos, sin, k_pages, v_pages, block_table, seq_lens, style,
                                    k_scales, v_scales, cu_seqlens)


def rope_qk_paged_hip_ctypes(q, k, v, cos, sin, k_pages, v_pages, block_table, seq_lens, style="neox",
                             k_scales=None, v_scales=None, cu_seqlens=None) -> torch.Tensor:
    fn = "rope_qk_paged_hip"
    index = gpu_index(q, fn)
    ref.refuse(fn, ref.cache_error(k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, cu_seqlens)
               or ref.write_error(q, k, v, cos, sin, k_pages, block_table, style, cu_seqlens))
    qv, kv, vv = _head_view(q), _head_view(k), _head_view(v)
    c, s, st = _table_stride(_table(cos, index), _table(sin, index))
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    cache = _cache(k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, cu_seqlens, _tokens(q))
    status = call(index, lib().ako_rope_qk_paged_fwd, qv.data_ptr(), kv.data_ptr(), vv.data_ptr(), c.data_ptr(),
                  s.data_ptr(), out.data_ptr(), ctypes.addressof(cache), q.shape[-2], _row_strides(qv),
                  _row_strides(kv), _row_strides(vv), c.shape[0], st, DT[q.dtype], DT[c.dtype],
                  _native.ROPE_STYLE_CODES[style], raw_stream(index))
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


def paged_attention_hip(q, k_pages, v_pages, block_table, seq_lens, scale=None, window=None, sinks=0,
                        k_scales=None, v_scales=None, cu_seqlens=None) -> torch.Tensor:
    """Attention of a step's rows over their sequences' pages."""
    fast = _native.torch_binding()
    if fast is not None:
        return fast.paged_attention(q, k_pages, v_pages, block_table, seq_lens, scale, window, sinks,
                                    k_scales, v_scales, cu_seqlens)
    return paged_attention_hip_ctypes(q, k_pages, v_pages, block_table, seq_lens, scale, window, sinks,
                                      k_scales, v_scales, cu_seqlens)


def paged_attention_hip_ctypes(q, k_pages, v_pages, block_table, seq_lens, scale=None, window=None, sinks=0,
                               k_scales=None, v_scales=None, cu_seqlens=None) -> torch.Tensor:
    fn = "paged_attention_hip"
    index = gpu_index(q, fn)
    ref.refuse(fn, ref.cache_error(k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, cu_seqlens)
               or ref.rows_error("q", q, -1, k_pages, block_table, cu_seqlens))
    scale = k_pages.shape[3] ** -0.5 if scale is None else scale
    ref.refuse(fn, ref.attention_error(q, k_pages, scale, window, sinks))
    qv = _head_view(q)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    cache = _cache(k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, cu_seqlens, _tokens(q))
    at, heads, dt = ctypes.addressof(cache), q.shape[-2], DT[q.dtype]
    need = lib().ako_paged_attention_workspace(at, heads, dt)
    space = torch.empty(need, dtype=torch.uint8, device=q.device) if need > 0 else None
    status = call(index, lib().ako_paged_attention_fwd, qv.data_ptr(), _row_strides(qv), out.data_ptr(), at, heads,
                  scale, window or 0, sinks, space.data_ptr() if space is not None else None, max(need, 0), dt,
                  raw_stream(index))
    if status:
        _native.check(status, fn)
    return out

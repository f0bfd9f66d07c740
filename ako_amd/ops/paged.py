"""Public operations on a paged key/value cache: write, read, attend.

They are called directly, not through the selector: the write changes the
caches in place, which the candidate contract rules out, and timing candidates
of the others would clone pools of many gigabytes. On a GPU they run the HIP
kernels (and raise if the library cannot be loaded, unless
``AKO_HIP_DISABLE=1``), on a CPU the plain operations of ``paged_ref``, where the
layout is described.

A step is described by three device tensors that all calls share, so that a
captured step can be replayed as they change: ``block_table (n, width)``,
``seq_lens (n,)`` (positions of each sequence with this step's tokens) and, for
packed rows, ``cu_seqlens (n + 1,)``, all int32.

    q = ako.rope_qk_paged(q, k, v, cos, sin, k_pages, v_pages, block_table, seq_lens)
    o = ako.paged_attention(q, k_pages, v_pages, block_table, seq_lens)
"""

from __future__ import annotations

import torch

from ako_amd.ops._registry import hip_disabled
from ako_amd.ops.paged_hip import paged_attention_hip, paged_read_hip, rope_qk_paged_hip
from ako_amd.ops.paged_ref import new_pages, paged_attention_ref, paged_read_ref, rope_qk_paged_ref


def rope_qk_paged(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    style: str = "neox",
    *,
    k_scales: torch.Tensor | None = None,
    v_scales: torch.Tensor | None = None,
    cu_seqlens: torch.Tensor | None = None,
) -> torch.Tensor:
    """RoPE of a step's q and k at their positions, with the rotated keys and the
    values stored in their sequences' pages; returns the rotated q.

    ``cos``/``sin`` hold the rows of positions 0, 1, .... With e4m3 pages
    (``k_scales``, ``v_scales``) keys and values are quantised as they are
    written, the keys straight from the 32-bit rotation. Padding rows of the
    result are zero; a row whose position has no page, or no table row, is not
    stored and its row of the result is NaN. The rows of a step must have slots
    of their own: pages that sequences share are full ones.
    """
    args = (q, k, v, cos, sin, k_pages, v_pages, block_table, seq_lens, style)
    if q.is_cuda and not hip_disabled():
        return rope_qk_paged_hip(*args, k_scales, v_scales, cu_seqlens)
    return rope_qk_paged_ref(*args, k_scales=k_scales, v_scales=v_scales, cu_seqlens=cu_seqlens)


def paged_read(
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    rows: int,
    dtype: torch.dtype | None = None,
    *,
    k_scales: torch.Tensor | None = None,
    v_scales: torch.Tensor | None = None,
    cu_seqlens: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """The stored keys and values of each sequence's last positions, as dense rows.

    Without ``cu_seqlens`` the last ``rows`` positions of every sequence, ``(batch,
    rows, kv_heads, head_dim)``; with it ``rows`` packed rows, ``(rows, kv_heads,
    head_dim)``, of which sequence ``i`` has ``cu_seqlens[i+1] - cu_seqlens[i]``.
    ``dtype`` is the pages' own, or for e4m3 pages the type to convert to. Rows
    that are padding or have no page are zero.
    """
    if k_pages.is_cuda and not hip_disabled():
        return paged_read_hip(k_pages, v_pages, block_table, seq_lens, rows, dtype, k_scales, v_scales, cu_seqlens)
    return paged_read_ref(k_pages, v_pages, block_table, seq_lens, rows, dtype, k_scales=k_scales,
                          v_scales=v_scales, cu_seqlens=cu_seqlens)


def paged_attention(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    *,
    k_scales: torch.Tensor | None = None,
    v_scales: torch.Tensor | None = None,
    cu_seqlens: torch.Tensor | None = None,
    scale: float | None = None,
    window: int | None = None,
    sinks: int = 0,
) -> torch.Tensor:
    """Attention of a step's tokens over what their sequences hold.

    Head ``h`` of q reads head ``h // (heads // kv_heads)`` of the cache. A row at
    position ``p`` sees the positions ``j <= p``; with ``window``, of those only
    ``j > p - window`` and the first ``sinks``. ``scale`` is ``head_dim ** -0.5``
    unless given. Rows that see nothing (padding) are zero, and what a row does
    not see has no influence on it, whatever is stored there. A row that sees keys, but
    whose scores are all -infinity, is NaN, as their softmax is; an infinity or NaN among
    the values that it sees makes its element of them that infinity or NaN (NaN also
    where an infinity's weight vanishes).
    """
    if q.is_cuda and not hip_disabled():
        return paged_attention_hip(q, k_pages, v_pages, block_table, seq_lens, scale, window, sinks,
                                   k_scales, v_scales, cu_seqlens)
    return paged_attention_ref(q, k_pages, v_pages, block_table, seq_lens, k_scales=k_scales, v_scales=v_scales,
                               cu_seqlens=cu_seqlens, scale=scale, window=window, sinks=sinks)


__all__ = ["new_pages", "paged_attention", "paged_read", "rope_qk_paged"]

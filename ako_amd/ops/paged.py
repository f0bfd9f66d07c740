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
from ako_amd.ops.paged_hip import (
    paged_attention_hip, paged_means_hip, paged_read_hip, paged_select_hip, rope_qk_paged_hip,
)
from ako_amd.ops.paged_ref import (
    new_pages, paged_attention_ref, paged_means_ref, paged_read_ref, paged_select_ref, rope_qk_paged_ref,
)


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
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
) -> torch.Tensor:
    """RoPE of a step's q and k at their positions, with the rotated keys and the
    values stored in their sequences' pages; returns the rotated q.

    With ``q_weight`` and ``k_weight``, ``(head_dim,)`` each, every head of q and k goes
    through its RMSNorm first, as in ``rmsnorm_rope_qk``.

    ``cos``/``sin`` hold the rows of positions 0, 1, .... With e4m3 pages
    (``k_scales``, ``v_scales``) keys and values are quantised as they are
    written, the keys straight from the rotation, which is in 32 bits (after norms,
    in 64 for the keys). Padding rows of the
    result are zero; a row whose position has no page, or no table row, is not
    stored and its row of the result is NaN. The rows of a step must have slots
    of their own: pages that sequences share are full ones.
    """
    args = (q, k, v, cos, sin, k_pages, v_pages, block_table, seq_lens, style)
    if q.is_cuda and not hip_disabled():
        return rope_qk_paged_hip(*args, k_scales, v_scales, cu_seqlens, q_weight, k_weight, eps)
    return rope_qk_paged_ref(*args, k_scales=k_scales, v_scales=v_scales, cu_seqlens=cu_seqlens, q_weight=q_weight,
                             k_weight=k_weight, eps=eps)


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


def paged_means(
    k_pages: torch.Tensor,
    k_means: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    rows: int,
    *,
    k_scales: torch.Tensor | None = None,
    cu_seqlens: torch.Tensor | None = None,
) -> torch.Tensor:
    """The means of the keys of every page that a step's rows have filled, into ``k_means
    (pages, kv_heads, head_dim)``, float32, which is returned.

    To be called after the step's write; ``rows`` is as in ``paged_read``. Pages that the step has not
    filled keep what stands there. ``paged_select`` reads the means of a sequence's full pages.
    """
    if k_pages.is_cuda and not hip_disabled():
        return paged_means_hip(k_pages, k_means, block_table, seq_lens, rows, k_scales, cu_seqlens)
    return paged_means_ref(k_pages, k_means, block_table, seq_lens, rows, k_scales=k_scales, cu_seqlens=cu_seqlens)


def paged_select(
    q: torch.Tensor,
    k_means: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    page_size: int,
    count: int,
    *,
    cu_seqlens: torch.Tensor | None = None,
    first: int = 1,
    last: int = 1,
) -> torch.Tensor:
    """The blocks (pages of a sequence, numbered from 0) that each row of q attends to, for each
    key head: int32 ``(..., kv_heads, count)``, ascending, -1 behind the last.

    A row may take the blocks up to its own. If they are more than ``count``, it takes the ``first``
    first and the ``last`` last of them, and of the others those whose mean key has the largest product with
    the sum of the queries that share the key head; of equal ones the lowest. Scores are formed in
    64 bits, and the order of their sums hangs on how many rows a call has: the choice is the same for
    every division of the work, but where two scores are closer than some 2^-50 of the size of their terms
    (equal means have equal scores in any order, and so have sums that 64 bits hold exactly). Every call
    repeats itself. Blocks without a page are not taken; padding rows take none.
    """
    if q.is_cuda and not hip_disabled():
        return paged_select_hip(q, k_means, block_table, seq_lens, page_size, count, first, last, cu_seqlens)
    return paged_select_ref(q, k_means, block_table, seq_lens, page_size, count, cu_seqlens=cu_seqlens, first=first, last=last)


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
    blocks: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of a step's tokens over what their sequences hold.

    Head ``h`` of q reads head ``h // (heads // kv_heads)`` of the cache. A row at
    position ``p`` sees the positions ``j <= p``; with ``window``, of those only
    ``j > p - window`` and the first ``sinks``. With ``blocks``, int32 ``(..., kv_heads, count)`` as
    ``paged_select`` gives it, a row sees of the positions ``j <= p`` those whose block ``j // page_size`` is
    listed for its token and key head: a set, in any order; a number below 0 or past the table
    names nothing. ``scale`` is ``head_dim ** -0.5``
    unless given. Rows that see nothing (padding) are zero, and what a row does
    not see has no influence on it, whatever is stored there. A row that sees keys, but
    whose scores are all -infinity, is NaN, as their softmax is; an infinity or NaN among
    the values that it sees makes its element of them that infinity or NaN (NaN also
    where an infinity's weight vanishes).
    """
    if q.is_cuda and not hip_disabled():
        return paged_attention_hip(q, k_pages, v_pages, block_table, seq_lens, scale, window, sinks,
                                   k_scales, v_scales, cu_seqlens, blocks)
    return paged_attention_ref(q, k_pages, v_pages, block_table, seq_lens, k_scales=k_scales, v_scales=v_scales,
                               cu_seqlens=cu_seqlens, scale=scale, window=window, sinks=sinks, blocks=blocks)


__all__ = ["new_pages", "paged_attention", "paged_means", "paged_read", "paged_select", "rope_qk_paged"]

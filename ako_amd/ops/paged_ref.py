"""Paged key/value cache and attention over it in plain PyTorch: the semantics
of the HIP operators, and what runs on a CPU.

Keys and values lie in pools of pages, ``(pages, kv_heads, page_size,
head_dim)``; position ``p`` of sequence ``i`` is slot ``p % page_size`` of page
``block_table[i, p // page_size]``, and an entry outside the pool is a page that
is not there. ``seq_lens[i]`` counts sequence ``i``'s positions with the step's
tokens. A step's rows are either ``(batch, seq, heads, head_dim)``, the last
``seq`` positions of every sequence, or packed ``(tokens, heads, head_dim)``
with ``cu_seqlens``: rows ``cu_seqlens[i] .. cu_seqlens[i+1]-1`` are the last
positions of sequence ``i``. Packed rows behind the last sequence, and rows whose
position would be negative, are padding.

Pages are of the rows' type, or ``torch.float8_e4m3fn`` with one E8M0 code
(``uint8`` c, standing for 2^(c-127), 255 for NaN) per 32 elements of a row.
"""

from __future__ import annotations

import math

import torch

from ako_amd.ops.rope_ref import ROPE_STYLES, rope_ref

ROW_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
E4M3 = torch.float8_e4m3fn
#: Elements that share a scale code.
SCALE_BLOCK = 32
MAX_HEAD_DIM = 256
#: A block table names fewer positions than this.
MAX_POSITIONS = 2**31 - 1 - 65536


def scale_codes(head_dim: int) -> int:
    return -(-head_dim // SCALE_BLOCK)


def new_pages(num_pages: int, kv_heads: int, page_size: int, head_dim: int, dtype: torch.dtype, *,
              device: torch.device | str = "cuda"):
    """``(k_pages, v_pages, k_scales, v_scales)`` of a new, zeroed pool; the scales
    are ``None`` unless ``dtype`` is ``torch.float8_e4m3fn``."""
    shape = (num_pages, kv_heads, page_size, head_dim)
    if dtype != E4M3:
        return torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device), None, None
    k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(E4M3) for _ in range(2))
    ks, vs = (torch.ones((*shape[:3], scale_codes(head_dim)), dtype=torch.uint8, device=device) for _ in range(2))
    return k, v, ks, vs


# ------------------------------------------------------------------ arguments --
def _on(t: torch.Tensor, like: torch.Tensor) -> bool:
    return t.device == like.device


def cache_error(k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, cu_seqlens) -> str | None:
    """The first thing wrong with a cache's tensors, or ``None``."""
    if k_pages.dim() != 4 or v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype:
        return (f"k_pages {tuple(k_pages.shape)} {k_pages.dtype} and v_pages {tuple(v_pages.shape)} {v_pages.dtype} "
                "must be (pages, kv_heads, page_size, head_dim) alike")
    head_dim = k_pages.shape[3]
    if head_dim < 16 or head_dim > MAX_HEAD_DIM or head_dim % 16:
        return f"head_dim must be a multiple of 16 up to {MAX_HEAD_DIM}, got {head_dim}"
    if k_pages.shape[1] < 1 or k_pages.shape[2] < 1:
        return "kv_heads and page_size must be at least 1"
    if k_pages.dtype not in (*ROW_DTYPES, E4M3):
        return f"pages must be float32/float16/bfloat16/float8_e4m3fn, got {k_pages.dtype}"
    if k_pages.stride(3) != 1 or v_pages.stride(3) != 1:
        return "page rows must be contiguous in head_dim"
    if k_pages.dtype == E4M3:
        want = (*k_pages.shape[:3], scale_codes(head_dim))
        for name, s in (("k_scales", k_scales), ("v_scales", v_scales)):
            if s is None or tuple(s.shape) != want or s.dtype != torch.uint8:
                return f"e4m3 pages need {name} of shape {want} and dtype uint8"
            if s.shape[3] > 1 and s.stride(3) != 1:
                return f"{name} must be contiguous in the last dimension"
    elif k_scales is not None or v_scales is not None:
        return "k_scales and v_scales are for float8_e4m3fn pages"
    if block_table.dim() != 2 or block_table.dtype != torch.int32:
        return "block_table must be a 2-D int32 tensor"
    if block_table.shape[1] > 1 and block_table.stride(1) != 1:
        return "block_table rows must be contiguous"
    n = block_table.shape[0]
    if block_table.shape[1] * k_pages.shape[2] > MAX_POSITIONS:
        return f"block_table names more than {MAX_POSITIONS} positions"
    if tuple(seq_lens.shape) != (n,) or seq_lens.dtype != torch.int32 or not seq_lens.is_contiguous():
        return f"seq_lens must be a contiguous int32 tensor of shape ({n},)"
    if cu_seqlens is not None and (tuple(cu_seqlens.shape) != (n + 1,) or cu_seqlens.dtype != torch.int32
                                   or not cu_seqlens.is_contiguous()):
        return f"cu_seqlens must be a contiguous int32 tensor of shape ({n + 1},)"
    for name, t in (("v_pages", v_pages), ("k_scales", k_scales), ("v_scales", v_scales),
                    ("block_table", block_table), ("seq_lens", seq_lens), ("cu_seqlens", cu_seqlens)):
        if t is not None and not _on(t, k_pages):
            return f"{name} must be on the device of the pages"
    return None


def rows_error(name, x, heads, k_pages, block_table, cu_seqlens) -> str | None:
    """The first thing wrong with a step's rows ``x``, or ``None``; ``heads`` -1 takes any number."""
    head_dim = k_pages.shape[3]
    if x.dim() != (4 if cu_seqlens is None else 3):
        return (f"{name} must be (batch, seq, heads, head_dim), or (tokens, heads, head_dim) with cu_seqlens, "
                f"got {tuple(x.shape)}")
    if x.shape[-1] != head_dim or (heads >= 0 and x.shape[-2] != heads):
        return f"{name} {tuple(x.shape)} does not match the pages {tuple(k_pages.shape)}"
    if cu_seqlens is None and x.shape[0] != block_table.shape[0]:
        return f"{name} has {x.shape[0]} sequences, the block table {block_table.shape[0]}"
    if x.dtype not in ROW_DTYPES:
        return f"{name} must be float32/float16/bfloat16, got {x.dtype}"
    if k_pages.dtype not in (x.dtype, E4M3):
        return f"{name} is {x.dtype}, the pages {k_pages.dtype}"
    if not _on(x, k_pages):
        return f"{name} must be on the device of the pages"
    return None


def attention_error(q, k_pages, scale, window, sinks) -> str | None:
    if q.shape[-2] % k_pages.shape[1]:
        return f"{q.shape[-2]} query heads are no multiple of {k_pages.shape[1]} key heads"
    if not math.isfinite(scale):
        return f"scale must be finite, got {scale}"
    if (window is not None and window < 1) or sinks < 0:
        return f"window must be at least 1 (or None) and sinks at least 0, got {window} and {sinks}"
    return None


def write_error(q, k, v, cos, sin, k_pages, block_table, style, cu_seqlens) -> str | None:
    if style not in ROPE_STYLES:
        return f"Unknown RoPE style '{style}', expected one of {ROPE_STYLES}"
    for name, x, heads in (("q", q, -1), ("k", k, k_pages.shape[1]), ("v", v, k_pages.shape[1])):
        wrong = rows_error(name, x, heads, k_pages, block_table, cu_seqlens)
        if wrong:
            return wrong
        if x.dtype != q.dtype or x.shape[:-2] != q.shape[:-2]:
            return f"{name} {tuple(x.shape)} {x.dtype} does not match q {tuple(q.shape)} {q.dtype}"
    if cos.dim() != 2 or cos.shape[1] != k_pages.shape[3] // 2 or sin.shape != cos.shape:
        return f"tables must be (positions, {k_pages.shape[3] // 2}), got {tuple(cos.shape)} and {tuple(sin.shape)}"
    if not _on(cos, q) or not _on(sin, q):
        return "tables must be on the device of the pages"
    return None


def refuse(fn_name: str, *errors: str | None) -> None:
    for e in errors:
        if e:
            raise ValueError(f"{fn_name}: {e}")


# ------------------------------------------------------------------- semantics --
def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows as e4m3 and their scale codes: for each block of 32 elements the
    smallest code c >= 1 with |x| <= 448 * 2^(c-127) for its finite elements;
    infinities and NaN become NaN."""
    d = x.shape[-1]
    n = scale_codes(d)
    xb = torch.nn.functional.pad(x.float(), (0, n * SCALE_BLOCK - d)).unflatten(-1, (n, SCALE_BLOCK))
    finite = xb.isfinite()
    amax = xb.where(finite, xb.new_zeros(())).abs().amax(-1)
    mantissa, exponent = torch.frexp(amax)  # 448 = 0.875 * 2^9
    e = torch.where(mantissa > 0.875, exponent - 8, exponent - 9).clamp_(min=-126).masked_fill_(amax == 0, -126)
    y = torch.ldexp(xb, -e.unsqueeze(-1)).where(finite, xb.new_full((), float("nan")))
    return y.flatten(-2)[..., :d].to(E4M3), (e + 127).to(torch.uint8)


def dequantize_rows(q: torch.Tensor, codes: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """What e4m3 rows with scale codes stand for, in ``dtype``; code 255 is E8M0's NaN."""
    scale = torch.ldexp(torch.ones((), device=q.device), codes.int() - 127).masked_fill_(codes == 255, math.nan)
    return (q.float() * scale.repeat_interleave(SCALE_BLOCK, -1)[..., : q.shape[-1]]).to(dtype)


def row_places(tokens: int, seq_lens, cu_seqlens):
    """``(sequence, position)`` of every row; padding has position -1."""
    n = seq_lens.shape[0]
    row = torch.arange(tokens, device=seq_lens.device)
    if cu_seqlens is None:
        seq = tokens // n if n else 0
        s = row // max(seq, 1)
        pos = seq_lens.clamp(min=0).long()[s] - seq + row % max(seq, 1)
        return s, pos.clamp(min=-1)
    cu = cu_seqlens.long()
    s = torch.searchsorted(cu, row, right=True) - 1
    inside = (s >= 0) & (s < n)
    s = s.clamp(0, max(n - 1, 0))
    if not n:
        return s, torch.full_like(row, -1)
    pos = seq_lens.clamp(min=0).long()[s] - (cu[s + 1] - row)
    return s, torch.where(inside, pos, -1).clamp(min=-1)


def row_slots(s, pos, block_table, page_size: int, num_pages: int):
    """``(page, slot)`` of every row, page -1 where there is none."""
    width = block_table.shape[1]
    if not width or not block_table.shape[0]:
        return torch.full_like(pos, -1), torch.zeros_like(pos)
    at = pos.clamp(min=0) // page_size
    page = block_table.long()[s, at.clamp(max=width - 1)]
    there = (pos >= 0) & (at < width) & (page >= 0) & (page < num_pages)
    return torch.where(there, page, -1), pos.clamp(min=0) % page_size


def _bytes(t: torch.Tensor) -> torch.Tensor:
    return t.view(torch.uint8) if t.dtype == E4M3 else t


def _rows(pages, codes, page, slot, dtype) -> torch.Tensor:
    """Rows ``(n, kv_heads, head_dim)`` at pages and slots."""
    x = _bytes(pages)[page, :, slot].view(pages.dtype)
    return x if codes is None else dequantize_rows(x, codes[page, :, slot], dtype)


def rope_qk_paged_ref(q, k, v, cos, sin, k_pages, v_pages, block_table, seq_lens, style="neox", *,
                      k_scales=None, v_scales=None, cu_seqlens=None) -> torch.Tensor:
    refuse("rope_qk_paged", cache_error(k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, cu_seqlens)
           or write_error(q, k, v, cos, sin, k_pages, block_table, style, cu_seqlens))
    num_pages, kv_heads, page_size, head_dim = k_pages.shape
    q2, k2, v2 = (x.flatten(0, -3) for x in (q, k, v))
    s, pos = row_places(q2.shape[0], seq_lens, cu_seqlens)
    page, slot = row_slots(s, pos, block_table, page_size, num_pages)
    page = torch.where(pos < cos.shape[0], page, -1)
    row = pos.clamp(0, max(cos.shape[0] - 1, 0))
    at = page >= 0
    out = torch.full_like(q2, float("nan")).masked_fill(pos.lt(0)[:, None, None], 0.0)
    if bool(at.any()):
        c, n, page, slot = cos[row[at]], sin[row[at]], page[at], slot[at]
        out[at] = rope_ref(q2[at][None], c, n, style)[0]
        # One rounding to 8 bits: the rotated keys are not rounded to the rows' type first.
        kr = rope_ref((k2[at] if k_scales is None else k2[at].float())[None], c, n, style)[0]
        if k_scales is None:
            k_pages[page, :, slot], v_pages[page, :, slot] = kr, v2[at]
        else:
            for pages, codes, x in ((k_pages, k_scales, kr), (v_pages, v_scales, v2[at])):
                b, e = quantize_rows(x)
                pages.view(torch.uint8)[page, :, slot] = b.view(torch.uint8)
                codes[page, :, slot] = e
    return out.view(q.shape)


def paged_read_ref(k_pages, v_pages, block_table, seq_lens, rows, dtype=None, *, k_scales=None, v_scales=None,
                   cu_seqlens=None) -> tuple[torch.Tensor, torch.Tensor]:
    refuse("paged_read", cache_error(k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, cu_seqlens),
           read_error(k_pages, rows, dtype))
    dtype = k_pages.dtype if dtype is None else dtype
    num_pages, kv_heads, page_size, head_dim = k_pages.shape
    n = block_table.shape[0]
    lead = (rows,) if cu_seqlens is not None else (n, rows)
    tokens = rows if cu_seqlens is not None else n * rows
    s, pos = row_places(tokens, seq_lens, cu_seqlens)
    page, slot = row_slots(s, pos, block_table, page_size, num_pages)
    at = page >= 0
    out = []
    for pages, codes in ((k_pages, k_scales), (v_pages, v_scales)):
        x = torch.zeros(tokens, kv_heads, head_dim, dtype=dtype, device=pages.device)
        x[at] = _rows(pages, codes, page[at], slot[at], dtype)
        out.append(x.view(*lead, kv_heads, head_dim))
    return out[0], out[1]


def read_error(k_pages, rows, dtype) -> str | None:
    if rows < 0:
        return f"rows must be at least 0, got {rows}"
    if (k_pages.dtype if dtype is None else dtype) not in ROW_DTYPES:
        return f"dtype must be float32/float16/bfloat16, got {dtype if dtype is not None else k_pages.dtype}"
    if dtype is not None and k_pages.dtype not in (dtype, E4M3):
        return f"dtype is {dtype}, the pages {k_pages.dtype}"
    return None


def paged_attention_ref(q, k_pages, v_pages, block_table, seq_lens, *, k_scales=None, v_scales=None,
                        cu_seqlens=None, scale=None, window=None, sinks=0) -> torch.Tensor:
    """Sequence by sequence, in 32 bits (64 for 64-bit arithmetic checks is the tests' own)."""
    refuse("paged_attention", cache_error(k_pages, v_pages, k_scales, v_scales, block_table, seq_lens, cu_seqlens)
           or rows_error("q", q, -1, k_pages, block_table, cu_seqlens))
    scale = k_pages.shape[3] ** -0.5 if scale is None else scale
    refuse("paged_attention", attention_error(q, k_pages, scale, window, sinks))
    num_pages, kv_heads, page_size, head_dim = k_pages.shape
    heads = q.shape[-2]
    q2 = q.flatten(0, -3)
    out = torch.zeros_like(q2, memory_format=torch.contiguous_format)
    s, pos = row_places(q2.shape[0], seq_lens, cu_seqlens)
    for i in range(block_table.shape[0]):
        rows = torch.nonzero((s == i) & (pos >= 0)).flatten()
        if not rows.numel() or not block_table.shape[1]:
            continue
        key = torch.arange(min(int(pos[rows].max()) + 1, block_table.shape[1] * page_size), device=q.device)
        page, slot = row_slots(torch.full_like(key, i), key, block_table, page_size, num_pages)
        key, page, slot = key[page >= 0], page[page >= 0], slot[page >= 0]
        kk = _rows(k_pages, k_scales, page, slot, q.dtype).float().repeat_interleave(heads // kv_heads, 1)
        vv = _rows(v_pages, v_scales, page, slot, q.dtype).float().repeat_interleave(heads // kv_heads, 1)
        at = pos[rows][:, None]
        seen = key <= at
        if window is not None:
            seen &= (key > at - window) | (key < sinks)
        score = torch.einsum("thd,jhd->htj", q2[rows].float(), kk) * scale
        score = score.masked_fill(~seen, float("-inf"))
        some = seen.any(-1)
        p = torch.softmax(score[:, some], -1)
        if bool(vv.isfinite().all()):
            o = torch.einsum("htj,jhd->thd", p, vv)
        else:  # a value that a row does not see must not reach it, not even as 0 * inf
            o = torch.where(seen[some][None, :, :, None], p[..., None] * vv.transpose(0, 1)[:, None], 0.0).sum(2).transpose(0, 1)
        out[rows[some]] = o.to(q.dtype)
    return out.view(q.shape)

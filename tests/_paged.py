"""Paged-cache test inputs, and the operators in 64 bits written from their definitions."""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

E4M3 = torch.float8_e4m3fn
U32 = 2.0 ** -24  # half a step of float32, relative


@dataclass
class Step:
    """A pool, its block table and one step's rows."""

    q: torch.Tensor
    k: torch.Tensor
    v: torch.Tensor
    k_pages: torch.Tensor
    v_pages: torch.Tensor
    k_scales: torch.Tensor | None
    v_scales: torch.Tensor | None
    table: torch.Tensor
    lens: torch.Tensor
    cu: torch.Tensor | None
    held: list[int]
    news: list[int]

    @property
    def where(self):
        return self.k_pages, self.v_pages, self.table, self.lens

    @property
    def kw(self):
        return {"k_scales": self.k_scales, "v_scales": self.v_scales, "cu_seqlens": self.cu}

    @property
    def rows(self) -> int:
        return self.q.shape[0] if self.cu is not None else self.q.shape[1]


def pages_of(shape, dtype, layout: str, device: str):
    """Zeroed k and v pools of a logical ``(pages, heads, slots, dim)`` shape."""
    n, h, p, d = shape
    raw = torch.uint8 if dtype == E4M3 else dtype
    if layout == "heads":
        k, v = (torch.zeros(n, h, p, d, dtype=raw, device=device) for _ in range(2))
    elif layout == "tokens":
        k, v = (torch.zeros(n, p, h, d, dtype=raw, device=device).transpose(1, 2) for _ in range(2))
    elif layout == "pair":  # keys and values of a page in one block
        both = torch.zeros(n, 2, h, p, d, dtype=raw, device=device)
        k, v = both[:, 0], both[:, 1]
    else:  # "odd": rows that start anywhere
        k, v = (torch.zeros(n * h * p * (d + 3) + 5, dtype=raw, device=device)[5:].view(n, h, p, d + 3)[..., :d]
                for _ in range(2))
    return (k.view(E4M3), v.view(E4M3)) if dtype == E4M3 else (k, v)


def step(held, news, *, heads=4, kv_heads=2, head_dim=64, page=16, dtype=torch.float32, mx=False, packed=False,
         pad_rows=0, layout="heads", device="cpu", seed=0, spare=3, width=None, fused=False, q_scale=1.5) -> Step:
    """``held``: positions per sequence with the step's; ``news``: its rows per sequence (all alike
    unless packed). Stored rows are random; slots and pages that no sequence holds are NaN."""
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    n = len(held)
    per = [max(0, -(-x // page)) for x in held]
    pool = sum(per) + spare
    order = torch.randperm(pool, generator=g)[: sum(per)]
    width = max(per + [1]) if width is None else width
    table = torch.full((n, width), -1, dtype=torch.int32)
    at = 0
    for i, m in enumerate(per):
        table[i, : min(m, width)] = order[at:at + m][:width].int()
        at += m
    pdt = E4M3 if mx else dtype
    k_pages, v_pages = pages_of((pool, kv_heads, page, head_dim), pdt, layout, device)
    live = torch.zeros(pool, page, dtype=torch.bool)
    for i, m in enumerate(held):
        for j in range(per[i]):
            if j < width:
                live[table[i, j], : min(page, m - j * page)] = True
    live = live[:, None, :, None].to(device)
    x = [(rnd(pool, kv_heads, page, head_dim) * s + b).to(device) for s, b in ((1.0, 0.0), (1.0, 0.25))]
    if mx:
        codes = -(-head_dim // 32)
        scales = [torch.randint(122, 130, (pool, kv_heads, page, codes), generator=g, dtype=torch.uint8).to(device)
                  for _ in range(2)]
        for t, a in zip((k_pages, v_pages), x):
            raw = (a * 16).to(E4M3).view(torch.uint8)
            t.view(torch.uint8).copy_(torch.where(live, raw, torch.full_like(raw, 0x7F)))
    else:
        scales = [None, None]
        for t, a in zip((k_pages, v_pages), x):
            t.copy_(torch.where(live, a, torch.full_like(a, math.nan)).to(dtype))
    tokens = sum(news) + pad_rows
    lead = (tokens,) if packed else (n, news[0] if n else 0)
    wide = [heads, kv_heads, kv_heads]
    scale = q_scale / (8 if mx else 1)
    if fused:
        row = (rnd(*lead, sum(wide) * head_dim) * scale).to(dtype).to(device)
        q, k, v = (t.unflatten(-1, (m, head_dim)) for t, m in zip(row.split([m * head_dim for m in wide], -1), wide))
    else:
        q, k, v = ((rnd(*lead, m, head_dim) * scale).to(dtype).to(device) for m in wide)
    cu = None
    if packed:
        cu = torch.tensor([0] + news).cumsum(0).int().to(device)
    return Step(q, k, v, k_pages, v_pages, *scales, table.to(device), torch.tensor(held, dtype=torch.int32, device=device),
                cu, list(held), list(news))


def stored(pages, codes, table, page_size, i, upto):
    """``(rows, present)`` of sequence i's first ``upto`` positions in 64 bits; absent rows are zero."""
    n, h, p, d = pages.shape
    j = torch.arange(upto, device=pages.device)
    col = j // page_size
    page = torch.full_like(j, -1)
    inside = col < table.shape[1]
    page[inside] = table[i].long()[col[inside]]
    there = (page >= 0) & (page < n)
    raw = pages.view(torch.uint8) if pages.dtype == E4M3 else pages
    x = raw[page.clamp(0, n - 1), :, j % page_size].view(pages.dtype).double()
    if codes is not None:
        c = codes[page.clamp(0, n - 1), :, j % page_size].double()
        x = x * torch.exp2(c - 127).repeat_interleave(32, -1)[..., :d]
    return torch.where(there[:, None, None], x, torch.zeros_like(x)), there


def places(s: Step):
    """``(row, sequence, position)`` of every row that is no padding."""
    out, t = [], 0
    for i, (n, m) in enumerate(zip(s.held, s.news)):
        for a in range(m):
            if n - m + a >= 0:
                out.append((t + a, i, n - m + a))
        t += m
    return out


def attention64(s: Step, *, scale=None, window=None, sinks=0):
    """``(out, bound)``: attention in 64 bits, and how far a result of q's type may be from it.

    With u half a step of the type: the result's rounding u |out|; the weights' rounding to
    the type for the products, u sum_j p_j |v_j| =: u A (float32: none, but the products' own
    U32 A); the scores' error e, which changes each weight by a factor of at most 1 + e
    and with it the sum and the total: 2 e A. e adds up the dot product's D + 4 roundings of
    terms |q_d k_d|, and for the exponent's argument, its maximum and exp2 4 roundings of the
    largest |score| and 2 of 1. The running sums add at most n / 16 + 64 roundings of A each.
    """
    q = s.q.flatten(0, -3).double()
    heads, d = q.shape[1:]
    kv_heads, page = s.k_pages.shape[1:3]
    scale = d ** -0.5 if scale is None else scale
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    u = torch.finfo(s.q.dtype).eps / 2
    t = 0
    for i, (n, m) in enumerate(zip(s.held, s.news)):
        n = min(n, s.table.shape[1] * page) if s.table.shape[1] else 0
        kk, there = stored(s.k_pages, s.k_scales, s.table, page, i, n)
        vv, _ = stored(s.v_pages, s.v_scales, s.table, page, i, n)
        at = (torch.arange(m, device=q.device) + s.held[i] - m)[:, None]
        key = torch.arange(n, device=q.device)
        seen = (key <= at) & there
        if window is not None:
            seen = seen & ((key > at - window) | (key < sinks))
        for h in range(heads if n and m else 0):
            x, y, z = q[t:t + m, h], kk[:, h * kv_heads // heads], vv[:, h * kv_heads // heads]
            score = (x @ y.T * scale).masked_fill(~seen, -math.inf)
            p = torch.softmax(score, -1).masked_fill(~seen, 0.0)  # rows that see nothing: zero
            size = (x.abs() @ y.abs().T * abs(scale)).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
            for r in range(m):  # what a row does not see stays out of its sums, whatever it is
                j = seen[r]
                out[t + r, h] = p[r, j] @ z[j]
                bound[t + r, h] = p[r, j] @ z[j].abs()
            e = U32 * ((d + 4) * size + 4 * size + 2)
            most = (u if u > U32 else 2 * U32) + 2 * e + 2 * U32 * (n / 16 + 64)
            bound[t:t + m, h] = bound[t:t + m, h] * most + u * out[t:t + m, h].abs()
        t += m
    tiny = torch.finfo(s.q.dtype).smallest_normal * torch.finfo(s.q.dtype).eps  # the subnormals' step
    return out.view(s.q.shape), bound.view(s.q.shape) + tiny


def assert_within(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, what="") -> None:
    """NaN and infinities in the same places, everything else within ``bound``."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in other places"
    ok = (got == want) | want.isnan() | ((got - want).abs() <= bound)
    if not bool(ok.all()):
        worst = ((got - want).abs() / bound).nan_to_num(0).max()
        raise AssertionError(f"{what}: {int((~ok).sum())} of {ok.numel()} values off, by up to {float(worst):.2f} bounds")


def e4m3_64(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Quantised rows in 64 bits: ``(values, codes)`` from the format's definition."""
    d = x.shape[-1]
    values, codes = torch.empty_like(x), []
    for b in range(0, d, 32):
        part = x[..., b:b + 32]
        finite = part.isfinite()
        amax = part.where(finite, torch.zeros_like(part)).abs().amax(-1, keepdim=True)
        e = torch.full_like(amax, -126)
        for c in range(-126, 121):  # the smallest exponent that holds the block
            e = torch.where(amax > 448 * 2.0 ** c, torch.full_like(e, c + 1), e)
        y = part.where(finite, torch.zeros_like(part)) / torch.exp2(e)
        _, ex = torch.frexp(y.abs().clamp(min=2.0 ** -6))
        unit = torch.exp2((ex - 4).double())
        values[..., b:b + 32] = (torch.round(y / unit) * unit * torch.exp2(e)).where(finite, torch.full_like(y, math.nan))
        codes.append(e + 127)
    return values, torch.cat(codes, -1)


def tables(rows: int, head_dim: int, device="cpu", dtype=torch.float32):
    from ako_amd.ops.rope_ref import build_rope_tables

    cos, sin = build_rope_tables(rows, head_dim)
    return cos.to(dtype).to(device), sin.to(dtype).to(device)

"""Infinities and NaN among stored values, and scale codes at the end of their range: they reach
every row that sees them, as the signed infinity or NaN, and no other row, whichever wavefront or
workgroup a row lies in."""

from __future__ import annotations

import math

import pytest
import torch

import ako_amd as ako
from tests._paged import E4M3, Step, attention64, step

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def results(s: Step, **opts):
    """The result with the kernel that the sizes choose and, on a GPU, with each by name."""
    yield "by size", ako.paged_attention(s.q, *s.where, **opts, **s.kw)
    if s.q.is_cuda:
        from ako_amd import _native

        for n, name in ((1, "rows"), (2, "chunk")):
            _native.set_tuning(3, 3, n)
            try:
                yield name, ako.paged_attention(s.q, *s.where, **opts, **s.kw)
            finally:
                _native.set_tuning(3, 3, 0)


def sees(s: Step, i: int, j: int, window=None, sinks=0) -> list[int]:
    """The rows of q that see key ``j`` of sequence ``i``."""
    first, n, m = sum(s.news[:i]), s.held[i], s.news[i]
    return [first + a for a in range(m)
            if j <= n - m + a and (window is None or j > n - m + a - window or j < sinks)]


def assert_same(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, what: str) -> None:
    """NaN where NaN is wanted, the signed infinity where that is, and everything else within ``bound``."""
    got, want = got.double(), want.double()
    finite = want.isfinite()
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in other places"
    assert torch.equal(got[want.isinf()], want[want.isinf()]), f"{what}: other infinities"
    off = (got - want).abs()[finite] / bound[finite]
    assert bool((off <= 1).all()), f"{what}: off by up to {float(off.max()):.2f} bounds"


def put(s: Step, wanted: torch.Tensor, i: int, j: int, kv_head: int, e: int, value: float, **opts) -> None:
    """Stores ``value`` as element ``e`` of key ``j``'s row of V, and in ``wanted`` for the rows that see it."""
    page, kv_heads = s.v_pages.shape[2], s.v_pages.shape[1]
    group = s.q.shape[-2] // kv_heads
    s.v_pages[s.table[i, j // page], kv_head, j % page, e] = value
    at = wanted.flatten(0, -3)
    heads = slice(kv_head * group, (kv_head + 1) * group)
    rows = sees(s, i, j, **opts)
    at[rows, heads, e] += value  # two at one place: their sum, as in the formula


CASES = [  # held, new rows, packed, query heads of 2 key heads
    ([129], [129], False, 2), ([512], [512], False, 2), ([200, 166], [129, 129], False, 8),
    ([75, 230, 1, 150], [75, 193, 1, 120], True, 8),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("opts", [{}, {"window": 100, "sinks": 3}, {"window": 200}], ids=["causal", "sinks", "window"])
@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("dtype", DTYPES)
def test_values_that_are_not_finite_reach_every_row_that_sees_them(dtype, case: int, opts, device: str) -> None:
    held, news, packed, heads = CASES[case]
    for head_dim in (64, 256) if case == 0 else (64,):
        s = step(held, news, heads=heads, head_dim=head_dim, dtype=dtype, packed=packed, device=device, seed=case)
        want, bound = attention64(s, **opts)
        for i, n in enumerate(held):
            for e, (j, value) in enumerate(((0, math.nan), (10, math.inf), (37, -math.inf), (63, math.nan), (64, math.inf),
                                            (100, -math.inf), (127, math.inf), (128, math.nan), (n - 1, math.inf))):
                if j < n:
                    put(s, want, i, j, e % 2, 7 * e, value, **opts)
            if n > 20:  # two at one element: NaN where a row sees both
                put(s, want, i, 15, 0, 5, math.inf, **opts)
                put(s, want, i, 20, 0, 5, -math.inf, **opts)
        for name, out in results(s, **opts):
            assert_same(out, want, bound, f"{name}, heads of {head_dim}")


# ------------------------------------------------------------------- scale codes --
def element(byte: int, code: int) -> float:
    """What an e4m3 byte under an E8M0 code stands for: 255 is the format's NaN."""
    x = float(torch.tensor([byte], dtype=torch.uint8).view(E4M3).double())
    return math.nan if code == 255 else x * 2.0 ** (code - 127)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_byte_under_every_code_reads_as_the_format_says(dtype, device: str) -> None:
    pages = torch.arange(256, dtype=torch.uint8).repeat(256, 1, 1, 1).contiguous().to(device).view(E4M3)
    codes = torch.arange(256, dtype=torch.uint8).view(256, 1, 1, 1).repeat(1, 1, 1, 8).to(device)
    table = torch.arange(256, dtype=torch.int32, device=device).view(256, 1)
    lens = torch.ones(256, dtype=torch.int32, device=device)
    k, v = ako.paged_read(pages, pages, table, lens, 1, dtype, k_scales=codes, v_scales=codes)
    want = torch.tensor([[element(b, c) for b in range(256)] for c in range(256)], dtype=torch.float64)
    want = want.float().to(dtype)  # exact in 32 bits but for what is infinite there: one rounding
    for got in (k.cpu().view(256, 256), v.cpu().view(256, 256)):
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(7, 8, 9), want.nan_to_num(7, 8, 9))


def swap_out_page_0(s: Step) -> None:
    """Moves what page 0 holds to a page that no sequence has: absent pages are often read as the first."""
    free = min(set(range(1, s.k_pages.shape[0])) - set(s.table.flatten().tolist()))
    for t in (s.k_pages.view(torch.uint8), s.v_pages.view(torch.uint8), s.k_scales, s.v_scales):
        t[free] = t[0]
    s.table[s.table == 0] = free


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("code", [0, 134, 135, 246, 247, 254, 255])
@pytest.mark.parametrize("dtype", DTYPES)
def test_codes_of_what_a_row_does_not_see_do_not_matter(dtype, code: int, device: str) -> None:
    """Slots and pages that no sequence has, and keys outside every row's window, under any code."""
    for held, news, packed in (([170, 90], [1, 1], False), ([170, 140], [129, 129], False), ([170, 33, 140], [150, 1, 64], True)):
        for head_dim, page in ((64, 16), (48, 7)):
            s = step(held, news, heads=8, head_dim=head_dim, page=page, dtype=dtype, mx=True, packed=packed, device=device)
            swap_out_page_0(s)
            s.table[0, 12 // page] = -1  # a page that is not there
            opts = {"window": 160, "sinks": 2} if held[0] - news[0] > 160 else {}
            want, bound = attention64(s, **opts)
            live = torch.zeros(s.k_pages.shape[0], page, dtype=torch.bool)
            for i, n in enumerate(held):
                for j in range(n):
                    if s.table[i, j // page] >= 0 and sees(s, i, j, **opts):
                        live[s.table[i, j // page], j % page] = True
            dead = ~live[:, None, :, None].to(device)
            for byte in (0x00, 0x01, 0x7E, 0xFE):
                for pages, codes in ((s.k_pages, s.k_scales), (s.v_pages, s.v_scales)):
                    pages.view(torch.uint8).masked_fill_(dead, byte)
                    codes.masked_fill_(dead, code)
                for name, out in results(s, **opts):
                    assert_same(out, want, bound, f"{name}, {held}, heads of {head_dim}, byte {byte:#x}")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,code", [(dtype, code) for dtype in DTYPES
                                        for code in ((135, 247, 255) if dtype == torch.float16 else (247, 254, 255))])
def test_codes_past_the_types_range_reach_the_rows_that_see_their_keys(dtype, code: int, device: str) -> None:
    """448 and -448 in one block of a key's values, under a code that makes them infinite in the rows' type.
    A scale that keeps every weight far above 0, times which an infinity would be NaN."""
    heads, kv_heads, page = 4, 2, 16
    for j in (3, 70, 127):
        s = step([150], [150], heads=heads, kv_heads=kv_heads, dtype=dtype, mx=True, device=device, seed=j)
        at = s.table[0, j // page], 0, j % page
        s.v_pages.view(torch.uint8)[at] = 0
        want, bound = attention64(s, scale=0.01)
        for e, byte in ((32, 0x7E), (40, 0xFE)):
            s.v_pages.view(torch.uint8)[(*at, e)] = byte
            want[0, j:, : heads // kv_heads, e] = math.copysign(math.inf, element(byte, 127))
        s.v_scales[(*at, 1)] = code
        if code == 255:
            want[0, j:, : heads // kv_heads, 32:] = math.nan
        for name, out in results(s, scale=0.01):
            assert_same(out, want, bound, f"{name}, key {j}")


# -------------------------------------------------------------------------- write --
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("style", ["neox", "interleaved"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_q_and_other_slots_of_a_write_of_values_that_are_not_finite(dtype, style: str, mx: bool, device: str) -> None:
    """A rotation by nothing: q comes back as it was, whatever k and v hold beside it, and slots that the step
    does not write keep their bytes."""
    for head_dim in (64, 80):
        s = step([70, 9], [5, 5], dtype=dtype, mx=mx, head_dim=head_dim, device=device)
        top = torch.finfo(dtype).max
        for x in (s.k, s.v):
            x[0, 0], x[0, 1, 0, 3], x[0, 2, 1, 40], x[1, 3, 0, 5], x[1, 4] = 0.0, math.inf, math.nan, -math.inf, top
        s.q[0, 1], s.q[1, 2, 0] = torch.finfo(dtype).tiny, top
        cos = torch.ones(70, head_dim // 2, device=device)
        bits = {1: torch.uint8, 2: torch.int16, 4: torch.int32}
        raw = lambda t: t.view(bits[t.element_size()])  # noqa: E731
        pools = [t for t in (s.k_pages, s.v_pages, s.k_scales, s.v_scales) if t is not None]
        before = [raw(t).clone() for t in pools]
        out = ako.rope_qk_paged(s.q, s.k, s.v, cos, torch.zeros_like(cos), *s.where, style, **s.kw)
        assert torch.equal(out, s.q)
        page = s.k_pages.shape[2]
        kept = torch.ones(s.k_pages.shape[0], 1, page, 1, dtype=torch.bool, device=device)
        for i, n in enumerate(s.held):
            for p in range(n - 5, n):
                kept[s.table[i, p // page], :, p % page] = False
        assert all(torch.equal(raw(t)[kept.expand(t.shape)], was[kept.expand(t.shape)]) for t, was in zip(pools, before))


# ------------------------------------------------------------------ weights of zero --
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("keys", [0, 64])
@pytest.mark.parametrize("news", [1, 40])
@pytest.mark.parametrize("dtype", DTYPES)
def test_nan_under_a_score_of_minus_infinity_is_not_lost(dtype, news: int, keys: int, device: str) -> None:
    """0 times NaN is NaN in the formula, also where a wavefront or a part of the keys sees nothing but scores
    of -infinity: the last key alone in its tile, and stretches of whole tiles."""
    from ako_amd import _native

    for held, first, last in ((33, 32, 33), (65, 64, 65), (97, 96, 97), (129, 128, 129), (300, 64, 128), (700, 0, 600),
                              (700, 576, 700)):
        if held < news:
            continue
        s = step([held], [news], heads=4, page=16, dtype=dtype, device=device, seed=held)
        s.q[..., 0] = 1.0
        for j in range(first, last):
            s.k_pages[s.table[0, j // 16], :, j % 16, 0] = -math.inf
        for j, e in ((first, 3), (last - 1, 50)):
            s.v_pages[s.table[0, j // 16], :, j % 16, e] = math.nan
        want, bound = attention64(s)
        assert bool(want.isnan().any())
        _native.set_tuning(3, 2, keys)
        try:
            for name, out in results(s):
                assert_same(out, want, bound, f"{name}, {held} keys, {first} to {last}")
        finally:
            _native.set_tuning(3, 2, 0)

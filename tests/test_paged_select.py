"""Means of filled pages, and the choice of blocks by them, against the definitions in 64 bits:
page sizes, layouts, packed and padded rows, ties, absent pages, values that are not finite,
refusals, other streams, captured steps."""

from __future__ import annotations

import math

import pytest
import torch

import ako_amd as ako
from ako_amd import _native
from ako_amd.ops import paged_hip
from tests._paged import E4M3, U32, assert_within, places, step

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


# ---------------------------------------------------------------------------- means --
def means64(s):
    """{(page, …): mean} of the pages that the step fills, and how far 32 bits may be from it: each of
    the page's additions and the division half a step of the sum of magnitudes."""
    page = s.k_pages.shape[2]
    out = {}
    for _, i, p in places(s):
        if p % page == page - 1 and p // page < s.table.shape[1]:
            at = int(s.table[i, p // page])
            if 0 <= at < s.k_pages.shape[0]:
                raw = s.k_pages.view(torch.uint8) if s.k_scales is not None else s.k_pages
                x = raw[at].view(s.k_pages.dtype).double()
                if s.k_scales is not None:
                    x = x * torch.exp2(s.k_scales[at].double() - 127).repeat_interleave(32, -1)[..., : x.shape[-1]]
                out[at] = (x.sum(1) / page, x.abs().sum(1) / page * U32 * (page + 2))
    return out


def check_means(s, means=None) -> None:
    pages, kv_heads, _, d = s.k_pages.shape
    if means is None:
        means = torch.full((pages, kv_heads, d), 7.0, device=s.k_pages.device)
    before = means.clone()
    want = means64(s)
    got = ako.paged_means(s.k_pages, means, s.table, s.lens, s.rows, k_scales=s.k_scales, cu_seqlens=s.cu)
    assert got is means or got.data_ptr() == means.data_ptr()
    for at in range(pages):
        if at in want:
            assert_within(got[at], *want[at], f"page {at}")
        else:
            assert torch.equal(got[at], before[at])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_means_of_filled_pages(dtype, mx: bool, device: str) -> None:
    for i, d in enumerate([16, 32, 48, 64, 80, 96, 112, 128, 160, 192, 240, 256]):
        page = (1, 7, 16, 24, 64, 3)[i % 6]
        for held, news, packed in (([2 * page, 3 * page + 1, page], [1, 1, 1], False), ([5 * page, 3, 0, 2 * page + 2], [4 * page, 3, 0, page], True),
                                   ([40, 47], [33, 33], False), ([4, 2], [6, 6], False)):
            s = step(held, news, heads=2, kv_heads=2, head_dim=d, dtype=dtype, mx=mx, packed=packed, pad_rows=3 * packed, page=page,
                     device=device, seed=i, layout=("heads", "tokens", "pair", "odd")[i % 4])
            check_means(s)


@pytest.mark.parametrize("device", DEVICES)
def test_means_into_strided_memory_and_past_absent_pages(device: str) -> None:
    s = step([64, 65, 70, 63], [20, 20, 20, 20], page=16, device=device)
    s.table[1, 3], s.table[2, 3] = -1, 10 ** 6
    wide = torch.full((s.k_pages.shape[0], 2, 3, 70), 7.0, device=device)
    check_means(s, wide[:, :, 1, 5:69])
    assert (wide[:, :, 0] == 7).all() and (wide[:, :, 2] == 7).all() and (wide[..., :5] == 7).all() and (wide[..., 69:] == 7).all()
    s.k_pages[s.table[0, 3].long(), 0, 3, 5] = math.inf
    s.k_pages[s.table[0, 3].long(), 1, 9, 6] = math.nan
    means = torch.zeros(s.k_pages.shape[0], 2, 64, device=device)
    ako.paged_means(s.k_pages, means, s.table, s.lens, 20)
    got = means[s.table[0, 3].long()]
    assert got[0, 5] == math.inf and got[1, 6].isnan() and got.isfinite().sum() == 126
    assert ako.paged_means(s.k_pages, means.clone().fill_(1), s.table, s.lens, 0).eq(1).all()


# ---------------------------------------------------------------------------- choice --
def chosen64(q, means, table, pos, page, count, first, last):
    """``(blocks, clear)`` of one row of q (heads, d): a list for each key head, from the definition,
    and whether the scores around the last one taken are further apart than 64-bit sums may be off."""
    kv_heads = means.shape[1]
    group = q.shape[0] // kv_heads
    out, clear = [], True
    held = [b for b in range(min(pos // page + 1, len(table))) if 0 <= table[b] < means.shape[0]] if pos >= 0 else []
    limit = min(pos // page + 1, len(table))
    for h in range(kv_heads):
        if limit <= count:
            out.append(held)
            continue
        always = [b for b in held if b < first or b > pos // page - last]
        rest = [b for b in held if b not in set(always)]
        x = q[h * group:(h + 1) * group].double().sum(0)
        m = means[[table[b] for b in rest], h].double() if rest else torch.zeros(0, means.shape[2], dtype=torch.float64)
        score = [-math.inf if math.isnan(v) else v for v in (m * x).sum(-1).tolist()]
        want = count - len(always)
        order = sorted(range(len(rest)), key=lambda j: (-score[j], rest[j]))
        if 0 < want < len(order):
            size = float((m.abs() * q[h * group:(h + 1) * group].double().abs().sum(0)).sum(-1).nan_to_num(0, 0, 0).max())
            a, b = score[order[want - 1]], score[order[want]]
            clear &= a == b or not abs(a - b) < 2.0 ** -40 * size
        out.append(sorted(always + [rest[j] for j in order[:want]]))
    return out, clear


def check_select(s, count, first=1, last=1, means=None, ties=False, least_clear=0.999) -> torch.Tensor:
    pages, kv_heads, page, d = s.k_pages.shape
    dev = s.q.device
    if means is None:
        g = torch.Generator().manual_seed(count)
        means = torch.randn(pages, kv_heads, d, generator=g)
        if ties:
            means = means.sign() * (torch.arange(pages) % 3 - 1)[:, None, None]
        means = means.to(dev)
    got = ako.paged_select(s.q, means, s.table, s.lens, page, count, cu_seqlens=s.cu, first=first, last=last)
    assert got.shape == (*s.q.shape[:-2], kv_heads, count) and got.dtype == torch.int32
    rows, host = got.flatten(0, -3).tolist(), means.cpu()
    q, table = s.q.flatten(0, -3).cpu(), s.table.tolist()
    at = {t: (i, p) for t, i, p in places(s)}
    clear_rows = 0
    for t in range(q.shape[0]):
        i, p = at.get(t, (0, -1))
        want, clear = chosen64(q[t], host, table[i] if table else [], p, page, count, first, last)
        clear_rows += clear
        for h in range(kv_heads):
            if clear:
                assert rows[t][h] == want[h] + [-1] * (count - len(want[h])), (t, h, p)
    assert clear_rows >= least_clear * q.shape[0]
    return got


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_choice_by_score(dtype, device: str) -> None:
    for i, d in enumerate([16, 32, 48, 64, 80, 96, 112, 128, 160, 192, 240, 256]):
        heads, kv_heads = ((4, 2), (3, 3), (7, 1), (16, 2))[i % 4]
        page = (1, 3, 2, 5)[i % 4]
        for held, news, packed in (([61 * page, 17], [1, 1], False), ([50 * page, 3, 0, 25, 70], [20, 3, 0, 9, 17], True),
                                   ([40 * page, 33, 90], [21, 21, 21], False), ([4, 33 * page], [6, 6], False)):
            s = step(held, news, heads=heads, kv_heads=kv_heads, head_dim=d, dtype=dtype, packed=packed, pad_rows=3 * packed,
                     page=page, device=device, seed=i, fused=i % 2 == 1)
            for count, first, last in ((1, 0, 1), (5, 1, 1), (9, 2, 3), (64, 1, 1)):
                check_select(s, count, first, last)


@pytest.mark.parametrize("device", DEVICES)
def test_equal_scores_take_the_lowest_blocks(device: str) -> None:
    s = step([300, 77], [3, 3], page=2, device=device, heads=2, kv_heads=1, head_dim=16)
    got = check_select(s, 10, means=torch.zeros(s.k_pages.shape[0], 1, 16, device=device))
    assert got[0, 2, 0].tolist() == [0, 1, 2, 3, 4, 5, 6, 7, 8, 149]
    for count in (4, 33, 60):
        check_select(s, count, ties=True)
    low = torch.full((s.k_pages.shape[0], 1, 16), -3.0, device=device)
    low[s.table[0, 70].long()] = 0.0
    low[s.table[0, 71].long()] = -0.0
    s.q.fill_(1.0)
    got = check_select(s, 4, means=low)
    assert got[0, 2, 0].tolist() == [0, 70, 71, 149]


@pytest.mark.parametrize("device", DEVICES)
def test_absent_pages_and_odd_scores(device: str) -> None:
    s = step([200, 190], [2, 2], page=4, device=device, heads=2, kv_heads=2, head_dim=32)
    s.table[0, 7], s.table[0, 0], s.table[0, 49] = -1, 10 ** 6, -5  # the first and the own among them
    s.table[1, 3:40] = -1
    for count in (1, 2, 6, 30, 47, 48, 64):
        check_select(s, count, min(1, count - 1), 1)
    means = torch.randn(s.k_pages.shape[0], 2, 32, device=device)
    means[s.table[0, 20].long(), 0, 3] = math.nan
    means[s.table[0, 21].long(), 0] = math.inf
    s.q[0, 1, 0] = 1.0  # its sum of queries stays finite and positive
    got = ako.paged_select(s.q, means, s.table, s.lens, 4, 40)[0, 1]
    assert 20 not in got[0].tolist() and 21 in got[0].tolist()
    got = ako.paged_select(s.q, means, s.table, s.lens, 4, 47)[0, 1]
    assert 20 in got[0].tolist()  # NaN comes last, but before nothing
    s.q[0, 1, 1, 5] = math.nan  # every score of head 1 is NaN, all alike
    assert ako.paged_select(s.q, means, s.table, s.lens, 4, 5)[0, 1, 1].tolist() == [1, 2, 3, 4, 5]  # blocks 0 and 49 are absent


@pytest.mark.parametrize("device", DEVICES)
def test_no_rows_no_blocks_no_heads(device: str) -> None:
    s = step([0, 3], [4, 4], page=4, device=device)  # the first has no positions, the second three
    got = check_select(s, 3)
    assert (got[0] == -1).all() and got[1, 1:, :, 0].eq(0).all()
    means = torch.zeros(5, 2, 64, device=device)
    assert (ako.paged_select(s.q, means, s.table[:, :0].contiguous(), s.lens, 4, 3) == -1).all()
    assert (ako.paged_select(s.q, means[:0], s.table, s.lens, 4, 3) == -1).all()
    assert ako.paged_select(s.q[:, :0], means, s.table, s.lens, 4, 3).shape == (2, 0, 2, 3)
    assert ako.paged_select(s.q[:0], means, s.table[:0], s.lens[:0], 4, 3).shape == (0, 4, 2, 3)


def test_positions_past_the_table() -> None:
    s = step([40], [1], page=4, width=6, kv_heads=2)
    check_select(s, 3, 1, 2)  # its own block, and the one before it, lie past the table
    assert -1 not in ako.paged_select(s.q, torch.randn(*s.k_pages.shape[:2], 64), s.table, s.lens, 4, 5).tolist()[0][0][0]


# ------------------------------------------------------------------------- refusals --
def bad_means():
    return [("shape", dict(means=lambda m: m[:, :, :32]), "k_means must be a float32"), ("type", dict(means=lambda m: m.double()), "k_means must be a float32"),
            ("last", dict(means=lambda m: m.repeat_interleave(2, -1)[..., ::2]), "contiguous in the last"),
            ("rows", dict(rows=-1), "rows must be"), ("table", dict(table=lambda t: t.long()), "2-D int32"),
            ("lens", dict(lens=lambda t: t[:1]), "seq_lens must be")]


def bad_select():
    return [("means", dict(means=lambda m: m[0]), "k_means must be a float32"), ("means type", dict(means=lambda m: m.half()), "k_means must be a float32"),
            ("page", dict(page=0), "page_size must be"), ("count", dict(count=1), "count at least their sum"), ("first", dict(first=-1), "count at least their sum"),
            ("last", dict(last=0), "count at least their sum"), ("heads", dict(q=lambda q: q[:, :, :3]), "no multiple"),
            ("rows", dict(q=lambda q: q[0]), "q must be"), ("q type", dict(q=lambda q: q.double()), "q must be float32"),
            ("head size", dict(q=lambda q: q[..., :32]), "does not match the pages"), ("cu", dict(cu=torch.zeros(2, dtype=torch.int32)), "cu_seqlens must be"),
            ("sequences", dict(q=lambda q: q[:1]), "sequences"), ("table", dict(table=lambda t: t[0]), "2-D int32")]


def refused_means(fn, change, device):
    s = step([9, 17], [1, 1], device=device)
    a = dict(means=torch.zeros(*s.k_pages.shape[:2], 64, device=device), rows=1, table=s.table, lens=s.lens)
    for k, f in change.items():
        a[k] = f(a[k]) if callable(f) else f
    return lambda: fn(s.k_pages, a["means"], a["table"], a["lens"], a["rows"], None, None)


def refused_select(fn, change, device):
    s = step([9, 17], [1, 1], device=device)
    a = dict(q=s.q, means=torch.zeros(*s.k_pages.shape[:2], 64, device=device), table=s.table, lens=s.lens, page=16, count=2, first=1,
             last=1, cu=None)
    for k, f in change.items():
        a[k] = f(a[k]) if callable(f) else f.to(device) if torch.is_tensor(f) else f
    return lambda: fn(a["q"], a["means"], a["table"], a["lens"], a["page"], a["count"], a["first"], a["last"], a["cu"])


def public_means(p, m, t, n, r, ks, cu):
    return ako.paged_means(p, m, t, n, r, k_scales=ks, cu_seqlens=cu)


def public_select(q, m, t, n, page, count, first, last, cu):
    return ako.paged_select(q, m, t, n, page, count, first=first, last=last, cu_seqlens=cu)


@pytest.mark.parametrize("name,change,message", bad_means())
def test_means_refusals(name, change, message) -> None:
    with pytest.raises(ValueError, match=message):
        refused_means(public_means, change, "cpu")()


@pytest.mark.parametrize("name,change,message", bad_select())
def test_select_refusals(name, change, message) -> None:
    with pytest.raises(ValueError, match=message):
        refused_select(public_select, change, "cpu")()


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")
def test_both_bindings_alike() -> None:
    fast = _native.torch_binding()
    for bad, refused, fns in ((bad_means(), refused_means, (fast.paged_means, paged_hip.paged_means_hip_ctypes)),
                              (bad_select(), refused_select, (fast.paged_select, paged_hip.paged_select_hip_ctypes))):
        for _, change, message in bad:
            said = []
            for fn in fns:
                with pytest.raises(ValueError, match=message) as e:
                    refused(fn, change, "cuda")()
                said.append(str(e.value))
            assert said[0] == said[1]
    s = step([90, 170], [11, 11], device="cuda", mx=True, dtype=torch.bfloat16, page=8)
    outs = []
    for suffix, m in (("", fast), ("_hip_ctypes", paged_hip)):
        means = torch.zeros(*s.k_pages.shape[:2], 64, device="cuda")
        getattr(m, "paged_means" + suffix)(s.k_pages, means, s.table, s.lens, 11, s.k_scales, None)
        outs.append((means, getattr(m, "paged_select" + suffix)(s.q, means, s.table, s.lens, 8, 6, 1, 2, None)))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1]) and outs[0][0].any()


# ----------------------------------------------------------- sizes, streams, graphs --
@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")
@pytest.mark.parametrize("blocks", [63, 64, 65, 255, 257, 1023, 1025, 4095, 4097, 5000])
def test_every_number_of_blocks(blocks: int) -> None:
    s = step([blocks, blocks // 2 + 1], [1, 1], page=1, heads=4, kv_heads=2, head_dim=32, device="cuda", dtype=torch.bfloat16)
    for count in (2, 17, 62, 300):
        check_select(s, count)
    check_select(s, 40, ties=True)


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")
def test_many_rows_agree_with_the_plain_form() -> None:
    g = torch.Generator(device="cuda").manual_seed(0)
    for n, new, packed in ((1, 700, False), (3, 100, False), (40, 3, False)):
        width, page = 150, 8
        held = [width * page - 5 * i for i in range(n)]
        table = torch.randperm(n * width, generator=g, device="cuda").int().view(n, width)
        lens = torch.tensor(held, dtype=torch.int32, device="cuda")
        q = torch.randn(n, new, 16, 128, generator=g, device="cuda").bfloat16()
        means = torch.randn(n * width, 4, 128, generator=g, device="cuda")
        from ako_amd.ops.paged_ref import paged_select_ref

        want = paged_select_ref(q, means, table, lens, page, 12, first=1, last=2)
        got = ako.paged_select(q, means, table, lens, page, 12, first=1, last=2)
        # Scores are some 11 apart at a standard deviation, 140 of them: two within 2^-40 of each other are 1 in 1e10.
        assert torch.equal(got, want)
        cu = torch.arange(0, n * new + 1, new, dtype=torch.int32, device="cuda")
        assert torch.equal(ako.paged_select(q.flatten(0, 1), means, table, lens, page, 12, first=1, last=2, cu_seqlens=cu),
                           got.flatten(0, 1))


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")
def test_streams_and_captured_steps() -> None:
    s = step([200, 180, 31], [1, 1, 1], page=4, device="cuda", width=64)
    s.table.copy_(torch.arange(3 * 64, device="cuda").view(3, 64))
    pool = torch.randn(3 * 64, 2, 4, 64, device="cuda")
    means = pool.mean(2)

    def run():
        ako.paged_means(pool, means, s.table, s.lens, 1)
        return ako.paged_select(s.q, means, s.table, s.lens, 4, 7)

    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run()
        graphs.append((g, out))
    for turn in range(6):
        s.lens.add_(1)
        s.q.copy_(torch.randn_like(s.q))
        pool.copy_(torch.randn_like(pool))
        before = means.clone()
        g, out = graphs[turn % 2]
        g.replay()
        got, filled = out.clone(), means.clone()
        torch.cuda.synchronize()
        means.copy_(before)
        assert torch.equal(run(), got) and torch.equal(means, filled)


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")
def test_pages_past_32_bit_offsets() -> None:
    pages, d = 70000, 256  # 70000 * 2 * 64 * 256 elements: past 2^31
    k = torch.zeros(pages, 2, 64, d, dtype=torch.float16, device="cuda")
    k[-1], k[-2] = 2.0, 1.0
    means = torch.zeros(pages, 2, d, device="cuda")
    table = torch.tensor([[0, pages - 2, 1, pages - 1, 2]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([5 * 64], dtype=torch.int32, device="cuda")
    ako.paged_means(k, means, table, lens, 5 * 64)
    assert means[-1].eq(2).all() and means[-2].eq(1).all() and not means[:-2].any()
    q = torch.ones(1, 1, 4, d, dtype=torch.float16, device="cuda")
    assert ako.paged_select(q, means, table, lens, 64, 3).flatten().tolist() == [0, 3, 4] * 2

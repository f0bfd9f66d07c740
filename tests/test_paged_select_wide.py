"""The block choice where a tile's scores do not fit in LDS: scored by one kernel into the workspace and chosen from there by
another, over slices of rows. Against the definition in 64 bits, at the widths where the forms of the second kernel
meet, with packed sequences in one tile, ties, absent pages, scores that are not finite, replays and other streams."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import ako_amd as ako
from ako_amd import _native
from ako_amd.ops import paged_hip
from ako_amd.ops import paged_ref as ref
from tests._paged import step
from tests.test_paged_select import check_select

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def workspace(q, means, table, lens, page: int, count: int, cu=None) -> int:
    """Bytes of scores that such a call holds outside LDS."""
    pages = ref.blocks_as_pages(means, page)
    cache = paged_hip._cache(pages, pages, None, None, table, lens, cu, paged_hip._tokens(q))
    dt = cache.page_dtype = paged_hip.DT[q.dtype]
    return _native.load().ako_paged_select_workspace(ctypes.addressof(cache), q.shape[-2], count, dt)


def held_outside(s, count: int) -> int:
    means = torch.empty(*s.k_pages.shape[:2], s.k_pages.shape[3], device="cuda")
    return workspace(s.q, means, s.table, s.lens, s.k_pages.shape[2], count, s.cu)


def check_wide(s, count: int, *args, **kw) -> torch.Tensor:
    assert held_outside(s, count) > 0
    return check_select(s, count, *args, **kw)


@pytest.mark.parametrize("width", [897, 1024, 1025, 4096, 4097])
def test_rows_of_one_sequence(width: int) -> None:
    """Tiles of 16 rows, the last of them short; every form of the second kernel."""
    for i, d in enumerate((64, 128, 256, 80)):
        s = step([width * 2], [23], page=2, heads=4, kv_heads=2, head_dim=d, dtype=DTYPES[i % 3], device="cuda", seed=i)
        assert s.table.shape[1] == width
        for count, first, last in ((3, 0, 1), (16, 1, 1), (70, 2, 5), (width - 1, 1, 1)):
            check_wide(s, count, first, last)
        check_wide(s, 40, ties=True)


@pytest.mark.parametrize("width", [14337, 20011])
def test_single_rows(width: int) -> None:
    s = step([width, width - 4000], [1, 1], page=1, heads=2, kv_heads=1, head_dim=32, dtype=torch.bfloat16, device="cuda")
    for count in (2, 65, 3000):
        check_wide(s, count)
    check_wide(s, 500, ties=True)
    assert held_outside(step([14336], [1], page=1, heads=2, kv_heads=1, head_dim=32, device="cuda"), 65) == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_sequences_share_tiles(dtype) -> None:
    """Rows of several sequences in a tile, among them rows with fewer blocks than are asked for, or none, and padding."""
    held, news = [2000, 31, 0, 1990, 700, 64, 1801], [21, 9, 0, 1, 40, 3, 19]
    s = step(held, news, page=2, heads=6, kv_heads=3, head_dim=96, dtype=dtype, packed=True, pad_rows=5, device="cuda")
    for count, first, last in ((4, 1, 1), (20, 3, 2), (33, 0, 1), (400, 1, 1)):
        got = check_wide(s, count, first, last)
        assert (got[-5:] == -1).all()


def test_absent_pages_and_odd_scores() -> None:
    s = step([1800, 1750], [18, 18], page=2, heads=2, kv_heads=2, head_dim=32, device="cuda")
    s.table[0, 7], s.table[0, 0], s.table[0, 899] = -1, 10 ** 6, -5  # the first and the last rows' own among them
    s.table[1, 3:870] = -1
    for count in (1, 2, 6, 30, 890):
        check_wide(s, count, min(1, count - 1), 1)
    means = torch.randn(s.k_pages.shape[0], 2, 32, device="cuda")
    means[s.table[0, 20].long(), 0, 3] = math.nan
    means[s.table[0, 21].long(), 0] = math.inf
    s.q[0, :, 0] = 1.0  # its sums of queries stay finite and positive
    got = ako.paged_select(s.q, means, s.table, s.lens, 2, 400)[0, :, 0]
    assert (got != 20).all() and (got == 21).any(-1).all()
    s.q[0, 1, 1, 5] = math.nan  # every score of that row and head is NaN, all alike: the lowest blocks that are there
    got = ako.paged_select(s.q, means, s.table, s.lens, 2, 5)
    assert got[0, 1, 1].tolist() == [1, 2, 3, 4, (1800 - 18 + 1) // 2]


def wide_call(rows: int, width: int, kv_heads: int, d: int, page: int = 4, whole: bool = False):
    """One long sequence's inputs; ``whole``: small whole numbers, whose sums are exact and often equal."""
    g = torch.Generator().manual_seed(rows + width)
    make = (lambda *n: torch.randint(-2, 3, n, generator=g).float()) if whole else lambda *n: torch.randn(*n, generator=g)
    q, means = make(1, rows, 2 * kv_heads, d).bfloat16(), make(width + 3, kv_heads, d)
    table = torch.randperm(width + 3, generator=g)[:width].int().view(1, width)
    return q.cuda(), means.cuda(), table.cuda(), torch.tensor([width * page - 1], dtype=torch.int32, device="cuda"), page


@pytest.mark.parametrize("whole", [False, True])
def test_slices_use_the_workspace_anew(whole: bool) -> None:
    """More than 64 MiB of scores: the second slice's rows are scored where the first's were."""
    call = wide_call(1500, 2000, 4, 128, whole=whole)
    need = workspace(*call[:4], call[4], 12)
    assert 0 < need < 1500 * 4 * 2000 * 8
    for count in (12, 100):
        want = ref.paged_select_ref(*(t.cpu() for t in call[:4]), call[4], count, first=1, last=2)
        assert torch.equal(ako.paged_select(*call, count, first=1, last=2).cpu(), want)


def test_both_forms_choose_alike() -> None:
    """The same rows alone, by the kernel that keeps their scores in LDS."""
    for whole in (False, True):
        q, means, table, lens, page = wide_call(37, 1500, 2, 64, whole=whole)
        got = ako.paged_select(q, means, table, lens, page, 24)
        assert workspace(q, means, table, lens, page, 24) > 0 == workspace(q[:, :1], means, table, lens, page, 24)
        for r in (0, 15, 16, 36):
            alone = ako.paged_select(q[:, r:r + 1], means, table, lens - (36 - r), page, 24)
            assert torch.equal(alone[0, 0], got[0, r])


def test_streams_and_replays() -> None:
    q, means, table, lens, page = wide_call(40, 1200, 2, 128)
    run = lambda: ako.paged_select(q, means, table, lens, page, 20)  # noqa: E731
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
        q.copy_(torch.randn_like(q))
        lens.sub_(3)
        want = run()
        g, out = graphs[turn % 2]
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)

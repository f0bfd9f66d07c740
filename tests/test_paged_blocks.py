"""Attention over listed blocks of a paged cache against the definition in 64 bits: head sizes, groups,
page sizes, lists of every kind, padding, absent pages, values that must not be seen, refusals,
other streams, captured steps, and a whole step: write, means, choice, attention."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import ako_amd as ako
from ako_amd import _native
from ako_amd.ops import paged_hip
from tests._paged import U32, assert_within, attention64, step, stored, tables

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def blocks64(s, blocks, scale=None):
    """``(out, bound)`` in 64 bits; the bound is attention64's, whose derivation holds for any set of keys."""
    q = s.q.flatten(0, -3).double()
    heads, d = q.shape[1:]
    kv_heads, page = s.k_pages.shape[1:3]
    scale = d ** -0.5 if scale is None else scale
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    u = torch.finfo(s.q.dtype).eps / 2
    lists, t = blocks.flatten(0, -3).tolist(), 0
    for i, (n, m) in enumerate(zip(s.held, s.news)):
        n = min(n, s.table.shape[1] * page) if s.table.shape[1] else 0
        kk, there = stored(s.k_pages, s.k_scales, s.table, page, i, n)
        vv, _ = stored(s.v_pages, s.v_scales, s.table, page, i, n)
        key = torch.arange(n, device=q.device)
        for r in range(m if n else 0):
            pos = s.held[i] - m + r
            for g in range(kv_heads):
                taken = torch.tensor(sorted({b for b in lists[t + r][g] if b >= 0}), device=q.device, dtype=torch.long)
                j = torch.nonzero((key <= pos) & there & torch.isin(key // page, taken)).flatten()
                if not j.numel():
                    continue
                for h in range(g * heads // kv_heads, (g + 1) * heads // kv_heads):
                    x, y, z = q[t + r, h], kk[j, g], vv[j, g]
                    p = torch.softmax(y @ x * scale, -1)
                    size = float((y.abs() @ x.abs() * abs(scale)).max())
                    e = U32 * ((d + 4) * size + 4 * size + 2)
                    most = (u if u > U32 else 2 * U32) + 2 * e + 2 * U32 * (n / 16 + 64)
                    out[t + r, h] = p @ z
                    bound[t + r, h] = (p @ z.abs()) * most + u * out[t + r, h].abs()
        t += m
    tiny = torch.finfo(s.q.dtype).smallest_normal * torch.finfo(s.q.dtype).eps
    return out.view(s.q.shape), bound.view(s.q.shape) + tiny


def lists(s, count, kind="mixed", seed=0):
    """Lists for every row and key head: own and first blocks, random ones, in any order, some twice, some
    outside the table, some empty."""
    g = torch.Generator().manual_seed(seed)
    shape = (*s.q.shape[:-2], s.k_pages.shape[1], count)
    width = max(1, s.table.shape[1])
    b = torch.randint(0, width, shape, generator=g)
    if kind == "mixed":
        odd = torch.rand(shape, generator=g)
        b = torch.where(odd < 0.15, -1, b)
        b = torch.where(odd > 0.9, width + torch.randint(0, 10 ** 9, shape, generator=g), b)
        b[..., 0] = 0
        flat = b.view(-1, count)
        flat[::5] = -7  # nothing at all
    return b.int().to(s.q.device)


def check(s, blocks, what="", **opts) -> torch.Tensor:
    got = ako.paged_attention(s.q, *s.where, blocks=blocks, **opts, **s.kw)
    assert_within(got, *blocks64(s, blocks, **opts), what)
    return got


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [16, 48, 64, 80, 128, 160, 256])
def test_head_sizes(d: int, dtype, mx: bool, device: str) -> None:
    for i, (held, news, packed) in enumerate((([130, 61], [1, 1], False), ([95, 70], [9, 9], False), ([75, 40, 0, 30], [25, 1, 0, 12], True))):
        s = step(held, news, heads=4, kv_heads=2, head_dim=d, dtype=dtype, mx=mx, packed=packed, pad_rows=2 * packed,
                 page=(16, 7, 32)[i], device=device, seed=d + i, layout=("heads", "tokens", "odd")[i])
        check(s, lists(s, 5, seed=i), f"{held} {news}")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (5, 1), (8, 1), (16, 1), (20, 1), (33, 1), (12, 4)])
def test_groups(heads: int, kv_heads: int, device: str) -> None:
    """Tiles of many tokens, of a part of one token's heads, and of parts of two."""
    for page in (3, 16):
        s = step([60, 33], [20, 20], heads=heads, kv_heads=kv_heads, head_dim=32, page=page, device=device, dtype=torch.bfloat16)
        check(s, lists(s, 4, seed=heads))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("page", [1, 2, 5, 15, 16, 17, 31, 32, 33, 48, 64, 100])
def test_page_sizes_and_lengths(page: int, device: str) -> None:
    for n in (1, page, page + 1, 3 * page - 1, 9 * page + 2):
        s = step([n, 4 * page], [1, 1], page=page, heads=4, kv_heads=2, head_dim=32, device=device, dtype=torch.float16, width=12)
        for count in (1, 2, 7, 30):
            check(s, lists(s, count, seed=n), f"{n} of {page}")


@pytest.mark.parametrize("device", DEVICES)
def test_all_blocks_are_the_whole_sequence(device: str) -> None:
    s = step([200, 133], [30, 30], page=16, heads=8, kv_heads=2, dtype=torch.bfloat16, device=device)
    every = torch.arange(13, dtype=torch.int32, device=device).flip(0).expand(2, 30, 2, 13)
    got = ako.paged_attention(s.q, *s.where, blocks=every, **s.kw)
    assert_within(got, *attention64(s))
    check(s, every, scale=-0.2)
    twice = torch.cat([every, every], -1)
    assert torch.equal(ako.paged_attention(s.q, *s.where, blocks=twice, **s.kw), got)


@pytest.mark.parametrize("device", DEVICES)
def test_rows_that_see_nothing_are_zero(device: str) -> None:
    s = step([0, 3, 40], [4, 4, 4], page=4, device=device)
    b = torch.full((3, 4, 2, 3), -1, dtype=torch.int32, device=device)
    assert not ako.paged_attention(s.q, *s.where, blocks=b).any()
    b[...] = 9  # the third sequence's last block: only its rows see it
    got = check(s, b)
    assert not got[:2].any() and got[2].any(-1).all()
    s.table[2, 9] = -1
    assert not check(s, b).any()
    none = step([5], [2], page=4, device=device)
    b = torch.zeros(1, 2, 2, 2, dtype=torch.int32, device=device)
    assert not ako.paged_attention(none.q, none.k_pages[:0], none.v_pages[:0], none.table, none.lens, blocks=b).any()
    assert not ako.paged_attention(none.q, none.k_pages, none.v_pages, none.table[:, :0].contiguous(), none.lens, blocks=b).any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("mx", [False, True])
def test_values_that_a_row_does_not_see_do_not_reach_it(mx: bool, device: str) -> None:
    """Slots of blocks that others list, of blocks that nobody lists, and behind the last position, full of NaN."""
    s = step([70, 70], [6, 6], page=8, device=device, heads=4, kv_heads=2, mx=mx, dtype=torch.bfloat16)
    b = torch.tensor([0, 2, 8], dtype=torch.int32, device=device).repeat(2, 6, 2, 1)
    b[0, ::2] = torch.tensor([0, 3, 8], dtype=torch.int32, device=device)
    for block in (3, 5):
        for t in (s.k_pages, s.v_pages):
            (t.view(torch.uint8) if mx else t)[s.table[:, block].long()] = 0x7F if mx else math.nan
    got = ako.paged_attention(s.q, *s.where, blocks=b, **s.kw)
    assert got[0, ::2].isnan().all() and got[0, 1::2].isfinite().all() and got[1].isfinite().all()
    clean = b.clone()
    clean[0, ::2, :, 1] = 2
    want, bound = blocks64(s, clean)
    assert_within(got[0, 1::2], want[0, 1::2], bound[0, 1::2])
    assert_within(got[1], want[1], bound[1])
    if not mx:
        s = step([40], [4], page=8, device=device)
        s.v_pages[s.table[0, 4].long(), :, 6, 3] = math.inf  # position 38: seen by the last two rows
        b = torch.tensor([1, 4], dtype=torch.int32, device=device).repeat(1, 4, 2, 1)
        got = ako.paged_attention(s.q, *s.where, blocks=b)
        assert got[0, :2].isfinite().all() and (got[0, 2:, :, 3] == math.inf).all() and got[0, 2:].isfinite().sum() == 2 * 4 * 63
        s.k_pages[s.table[0, 1].long()] = 0.0
        s.k_pages[s.table[0, 1].long(), :, :, 0] = -math.inf
        s.q[...] = 1.0
        b[...] = 1
        assert ako.paged_attention(s.q, *s.where, blocks=b).isnan().all()  # scores of -infinity alone


def test_odd_indexes_are_survived() -> None:
    s = step([20, 30], [2, 2], page=4)
    b = torch.full((2, 2, 2, 4), 2 ** 31 - 1, dtype=torch.int32)
    b[..., 1], b[..., 2] = -2 ** 31, 7
    got = ako.paged_attention(s.q, *s.where, blocks=b)
    assert not got[0].any() and got[1].any()


# ------------------------------------------------------------------------- refusals --
def bad_blocks():
    good = torch.zeros(2, 1, 2, 3, dtype=torch.int32)
    return [(good.long(), {}, "blocks must be an int32"), (good[0], {}, "blocks must be an int32"), (good[:, :, :1], {}, "blocks must be an int32"),
            (good[..., :0], {}, "at least one number"), (good[:1], {}, "blocks must be an int32"), (good, {"window": 4}, "no room"),
            (good, {"sinks": 2}, "no room")]


@pytest.mark.parametrize("blocks,opts,message", bad_blocks(), ids=range(7))
def test_refusals(blocks, opts, message: str) -> None:
    s = step([9, 17], [1, 1])
    with pytest.raises(ValueError, match=message):
        ako.paged_attention(s.q, *s.where, blocks=blocks, **opts)


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")
def test_both_bindings_alike() -> None:
    fast = _native.torch_binding()
    for blocks, opts, message in bad_blocks():
        said = []
        for fn in (fast.paged_attention, paged_hip.paged_attention_hip_ctypes):
            s = step([9, 17], [1, 1], device="cuda")
            with pytest.raises(ValueError, match=message) as e:
                fn(s.q, *s.where, None, opts.get("window"), opts.get("sinks", 0), None, None, None, blocks.cuda())
            said.append(str(e.value))
        assert said[0] == said[1]
    s = step([900, 1700], [3, 3], device="cuda", dtype=torch.float16)
    with pytest.raises(ValueError, match="device of the pages"):
        ako.paged_attention(s.q, *s.where, blocks=lists(s, 40).cpu())
    b = lists(s, 40).repeat_interleave(2, -1)[..., ::2]
    a, c = (fn(s.q, *s.where, None, None, 0, None, None, None, b) for fn in (fast.paged_attention, paged_hip.paged_attention_hip_ctypes))
    assert torch.equal(a, c) and a.any()


def test_c_entries_refuse_what_they_cannot_do() -> None:
    if torch.cuda.is_available():
        pytest.skip("passes fake device addresses: runs only where no GPU is visible")
    from tests.test_paged_abi import F16, I3, INVALID, LENS, MIB, NO_DEVICE, OUT, Q, UNSUPPORTED, WS, cache

    lib = _native.load()
    blocks, means = 20 << 34, 21 << 34
    st, ms = I3(256, 256, 64), I3(128, 64, 0)

    def attend(c, count=4, at=blocks, ws=WS, size=None, dtype=F16):
        need = lib.ako_paged_attention_blocks_workspace(ctypes.addressof(c), 4, count, dtype)
        return lib.ako_paged_attention_blocks_fwd(Q, st, OUT, ctypes.addressof(c), 4, 0.1, at, count, ws, max(need, 0) if size is None else size, dtype, None)

    def select(c, q=Q, m=means, out=blocks, count=3, first=1, last=1, ws=WS, size=None, dtype=F16, mstr=ms):
        need = lib.ako_paged_select_workspace(ctypes.addressof(c), 4, count, dtype)
        return lib.ako_paged_select_fwd(ctypes.addressof(c), q, st, 4, m, mstr, out, count, first, last, ws, max(need, 0) if size is None else size, dtype, None)

    def mean(c, m=means, mstr=ms, dtype=F16):
        return lib.ako_paged_means_fwd(ctypes.addressof(c), m, mstr, dtype, None)

    long = cache(pages=64, width=64)
    assert attend(cache()) == attend(long, count=40) == select(cache()) == mean(cache()) == NO_DEVICE
    assert mean(cache(v_pages=None)) == select(cache(k_pages=None, v_pages=None)) == NO_DEVICE  # not used
    assert attend(cache(tokens=0)) == select(cache(tokens=0)) == mean(cache(tokens=0)) == 0
    for kw, m in ((dict(count=0), "count"), (dict(count=1 << 31), "count"), (dict(at=None), "null"), (dict(at=OUT), "overlaps")):
        assert attend(cache(), **kw) == INVALID and m in _native.last_error(), kw
    for kw in (dict(size=16), dict(ws=None), dict(ws=WS + 8)):
        assert attend(long, count=40, **kw) == INVALID and "workspace" in _native.last_error()
    assert attend(long, count=40, ws=blocks) == INVALID and "overlaps" in _native.last_error()
    assert attend(cache(), dtype=7) == select(cache(), dtype=7) == UNSUPPORTED
    assert lib.ako_paged_attention_blocks_workspace(ctypes.addressof(cache()), 4, 0, F16) == -1
    for kw, m in ((dict(q=None), "null"), (dict(m=None), "null"), (dict(out=None), "null"), (dict(mstr=None), "null"), (dict(count=0), "count"),
                  (dict(count=1), "first"), (dict(first=-1), "first"), (dict(last=0), "first"), (dict(out=Q), "overlap"), (dict(out=means), "overlap"),
                  (dict(out=LENS), "overlap"), (dict(mstr=I3(-1, 1, 0)), "negative")):
        assert select(cache(), **kw) == INVALID and m in _native.last_error(), kw
    for kw in (dict(size=16), dict(ws=None), dict(ws=WS + 8)):
        assert select(cache(pages=64, width=1 << 16), **kw) == INVALID and "workspace" in _native.last_error()
    assert lib.ako_paged_select_workspace(ctypes.addressof(long), 4, 3, F16) == 0  # a tile's scores fit in LDS
    assert select(cache(kv_heads=4, width=1 << 27, page=1), ws=WS) == INVALID and "2^28" in _native.last_error()
    assert lib.ako_paged_select_workspace(ctypes.addressof(cache(kv_heads=3)), 4, 3, F16) == -1
    for kw, m in ((dict(m=None), "null"), (dict(mstr=None), "null"), (dict(mstr=I3(64, 64, 0)), "rows of the means"), (dict(m=LENS), "overlap"),
                  (dict(mstr=I3(-1, 0, 0)), "negative")):
        assert mean(cache(), **kw) == INVALID and m in _native.last_error(), kw
    assert MIB


# --------------------------------------------------------------- sizes, streams, graphs --
@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")
@pytest.mark.parametrize("dtype,mx", [(torch.float16, False), (torch.bfloat16, True), (torch.float32, False)])
def test_long_tables_in_segments(dtype, mx: bool) -> None:
    """More blocks than a segment holds, lists that leave whole segments out, and parts that are joined."""
    for page, n, count in ((1, 5000, 300), (2, 9001, 700), (16, 40000, 60), (1, 70000, 9)):
        s = step([n, n // 3], [2, 2], page=page, heads=4, kv_heads=2, head_dim=64, dtype=dtype, mx=mx, device="cuda")
        b = lists(s, count, "plain", seed=n)
        check(s, b, f"{n} of {page}")
        b[..., : count // 2] = torch.arange(count // 2, device="cuda", dtype=torch.int32)
        b[1, ..., count // 2:] = n // page - 1 - torch.arange(count - count // 2, device="cuda", dtype=torch.int32)
        check(s, b, f"{n} of {page}, both ends")


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")
@pytest.mark.parametrize("count", [1, 3, 8, 16, 33, 64])
def test_parts(count: int) -> None:
    for batch in (1, 2, 30):
        held = [4000 - 37 * i for i in range(batch)]
        s = step(held, [1] * batch, page=64, heads=8, kv_heads=2, head_dim=128, dtype=torch.bfloat16, device="cuda")
        check(s, lists(s, count, "plain", seed=batch))
        assert torch.equal(*(ako.paged_attention(s.q, *s.where, blocks=lists(s, count), **s.kw) for _ in range(2)))


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")
def test_streams_and_captured_steps() -> None:
    s = step([1500, 900], [1, 1], page=16, heads=8, kv_heads=2, dtype=torch.float16, device="cuda", width=100, spare=120)
    s.table.copy_(torch.randperm(s.k_pages.shape[0], device="cuda")[:200].view(2, 100).int() if s.k_pages.shape[0] >= 200 else s.table)
    s.k_pages.copy_(torch.randn_like(s.k_pages, dtype=torch.float32))
    s.v_pages.copy_(torch.randn_like(s.v_pages, dtype=torch.float32))
    b = lists(s, 30)
    run = lambda: ako.paged_attention(s.q, *s.where, blocks=b, **s.kw)  # noqa: E731
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
        s.lens.add_(7)
        s.q.copy_(torch.randn_like(s.q))
        b.copy_(lists(s, 30, seed=turn))
        want = run()
        g, out = graphs[turn % 2]
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("mx", [False, True])
def test_a_whole_step(mx: bool, device: str) -> None:
    """A prompt in two chunks and single tokens: norm, rotate and store, means of what filled, choice, attention."""
    n, heads, kv_heads, d, page, count = 2, 4, 2, 32, 4, 4
    g = torch.Generator().manual_seed(11)
    kp, vp, ks, vs = ako.new_pages(n * 16, kv_heads, page, d, torch.float8_e4m3fn if mx else torch.float32, device=device)
    means = torch.zeros(n * 16, kv_heads, d, device=device)
    table = torch.randperm(n * 16, generator=g).int().view(n, 16).to(device)
    lens = torch.zeros(n, dtype=torch.int32, device=device)
    cos, sin = tables(64, d, device)
    w = torch.ones(d, device=device)
    held = 0
    for new in (21, 9, 1, 1, 1, 1, 1, 1):
        held += new
        lens.fill_(held)
        q, k, v = (torch.randn(n, new, h, d, generator=g).to(device) for h in (heads, kv_heads, kv_heads))
        where, sc = (kp, vp, table, lens), {"k_scales": ks, "v_scales": vs}
        q = ako.rope_qk_paged(q, k, v, cos, sin, *where, q_weight=w, k_weight=w, **sc)
        ako.paged_means(kp, means, table, lens, new, k_scales=ks)
        keys = ako.paged_read(*where, held, torch.float32, **sc)[0]
        for i in range(n):
            for b in range(held // page):
                mine = keys[i, b * page:(b + 1) * page].double()
                assert_within(means[table[i, b].long()], mine.mean(0), mine.abs().mean(0) * U32 * (page + 2))
        b = ako.paged_select(q, means, table, lens, page, count)
        assert (b[..., 0] == 0).all() and b.shape == (n, new, kv_heads, count)
        got = ako.paged_attention(q, *where, blocks=b, **sc)
        s = step([held] * n, [new] * n, heads=heads, kv_heads=kv_heads, head_dim=d, page=page, device=device)
        s.q, s.k_pages, s.v_pages, s.k_scales, s.v_scales, s.table, s.lens = q, kp, vp, ks, vs, table, lens
        assert_within(got, *blocks64(s, b))
        if held // page < count:
            assert_within(got, *attention64(s))

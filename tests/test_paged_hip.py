"""The paged-cache kernels on a GPU against the definitions in 64 bits: head sizes, types, page
sizes and layouts, lengths around every tile edge, windows, padding, absent pages, values that
must not be seen, other streams, captured steps, offsets past 32 bits."""

from __future__ import annotations

import math

import pytest
import torch

import ako_amd as ako
from ako_amd.ops import paged_hip
from tests._paged import E4M3, assert_within, attention64, step, stored, tables
from tests.test_paged_ref import bad_calls, check_write

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]
DEV = "cuda"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
HEAD_DIMS = [16, 32, 48, 64, 80, 96, 112, 128, 160, 192, 256]


def set_kernel(n: int) -> None:
    from ako_amd import _native

    _native.set_tuning(3, 3, n)


@pytest.fixture(params=["by size", "chunk"])
def kernel(request):
    """As the sizes choose, which for small cases is 16 rows per workgroup, and with 128."""
    set_kernel(2 if request.param == "chunk" else 0)
    yield
    set_kernel(0)


def attend(s, **opts):
    return ako.paged_attention(s.q, *s.where, **opts, **s.kw)


def check(s, what="", **opts) -> None:
    """Against 64 bits, with the kernel that the sizes choose and with that of long chunks."""
    want, bound = attention64(s, **opts)
    assert_within(attend(s, **opts), want, bound, what)
    set_kernel(2)
    try:
        assert_within(attend(s, **opts), want, bound, what + ", chunk")
    finally:
        set_kernel(0)


# ------------------------------------------------------------------------ write, read --
@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("style", ["neox", "interleaved"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_write_and_read_back(dtype, style: str, mx: bool) -> None:
    for i, d in enumerate(HEAD_DIMS):
        heads, kv_heads = ((4, 2), (3, 3), (7, 1))[i % 3]
        for held, news, packed in (([9, 30], [1, 1], False), ([12, 3, 0, 25, 70], [5, 3, 0, 9, 64], True),
                                   ([40, 33], [33, 33], False)):
            s = step(held, news, heads=heads, kv_heads=kv_heads, head_dim=d, dtype=dtype, mx=mx, packed=packed,
                     pad_rows=3 * packed, page=(1, 7, 16)[i % 3], device=DEV, seed=i,
                     layout=("heads", "tokens", "pair", "odd")[i % 4], fused=i % 2 == 1)
            cos, sin = tables(80, d, DEV, (torch.float32, dtype)[i % 2])
            before = [t.clone() for t in (s.k_pages, s.v_pages)]
            out = ako.rope_qk_paged(s.q, s.k, s.v, cos, sin, *s.where, style, **s.kw)
            check_write(s, out, cos, sin, style, before)


def test_write_of_values_the_format_cannot_hold() -> None:
    for dtype in DTYPES:
        s = step([70], [70], dtype=dtype, mx=True, head_dim=64, device=DEV)
        top = torch.finfo(dtype).max
        for x in (s.k, s.v):
            x[0, 0], x[0, 1, 0, 3], x[0, 2, 1, 40], x[0, 3, 0, 5] = 0.0, math.inf, math.nan, -math.inf
            x[0, 4], x[0, 5, 0, 0], x[0, 6] = 448.0, 450.0, torch.finfo(dtype).tiny
            x[0, 7, 0], x[0, 8, 1, 9] = top, top
        cos, sin = torch.ones(70, 32, device=DEV), torch.zeros(70, 32, device=DEV)
        before = [s.k_pages.clone(), s.v_pages.clone()]
        out = ako.rope_qk_paged(s.q, s.k, s.v, cos, sin, *s.where, **s.kw)
        # 0 * inf in the rotation turns the partner of an infinity into NaN: k is checked through v.
        k, v = ako.paged_read(*s.where, 70, torch.float32, **s.kw)
        from tests._paged import e4m3_64

        want = e4m3_64(s.v[0].double())[0]
        assert torch.equal(v[0].double().isnan(), want.isnan())
        assert torch.equal(v[0].double().nan_to_num(0, math.inf, -math.inf), want.float().double().nan_to_num(0, math.inf, -math.inf))
        assert torch.equal(k[0, 9:].double(), e4m3_64(s.k[0, 9:].double())[0])
        assert out.shape == s.q.shape and before[0].shape == s.k_pages.shape


def test_positions_without_a_slot() -> None:
    s = step([20, 6, 9], [1, 1, 1], page=4, device=DEV)
    s.table[2, 2] = -1
    cos, sin = tables(18, 64, DEV)
    before = [s.k_pages.clone(), s.v_pages.clone()]
    out = ako.rope_qk_paged(s.q, s.k, s.v, cos, sin, *s.where)
    assert out[0].isnan().all() and out[2].isnan().all() and torch.isfinite(out[1]).all()
    changed = (s.k_pages.nan_to_num(7) != before[0].nan_to_num(7)).any(-1).any(1).nonzero().tolist()
    assert changed == [[int(s.table[1, 1]), 1]]


# --------------------------------------------------------------------------- attention --
@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", HEAD_DIMS)
def test_head_sizes(d: int, dtype, mx: bool) -> None:
    for i, (held, news, packed) in enumerate((([130, 61], [1, 1], False), ([200, 90], [40, 40], False),
                                              ([75, 140, 30], [75, 1, 12], True))):
        s = step(held, news, heads=8, kv_heads=2, head_dim=d, dtype=dtype, mx=mx, packed=packed, page=16, device=DEV,
                 seed=d + i)
        check(s, f"{held} {news}")


LENGTHS = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300, 511, 513, 1025]


@pytest.mark.parametrize("page", [1, 7, 16, 24, 32, 64, 128])
@pytest.mark.parametrize("dtype,mx", [(torch.float16, False), (torch.bfloat16, True), (torch.float32, False)])
def test_single_tokens_at_every_length(dtype, mx: bool, page: int) -> None:
    for group in (1, 4, 8):
        s = step(LENGTHS, [1] * len(LENGTHS), heads=2 * group, kv_heads=2, head_dim=64, dtype=dtype, mx=mx, page=page,
                 device=DEV, seed=group)
        check(s, f"group {group}")


@pytest.mark.parametrize("page", [7, 16, 64])
@pytest.mark.parametrize("dtype,mx", [(torch.float16, False), (torch.float16, True), (torch.bfloat16, False),
                                      (torch.float32, True)])
def test_chunks_at_every_length(dtype, mx: bool, page: int) -> None:
    for group, news in ((1, [1, 2, 3, 16, 17, 33, 64, 65, 127, 128, 129, 200]), (4, [1, 4, 5, 8, 9, 31, 32, 33, 63, 150]),
                        (7, [1, 2, 3, 5, 18, 19, 40]), (32, [1, 2, 4, 5])):
        held = [n + (0, 1, 30, 64, 100)[i % 5] for i, n in enumerate(news)]
        s = step(held, news, heads=2 * group, kv_heads=2, head_dim=128, dtype=dtype, mx=mx, page=page, packed=True,
                 pad_rows=5, device=DEV, seed=group)
        check(s, f"group {group}")


@pytest.mark.parametrize("mx", [False, True])
def test_windows_and_sinks(mx: bool) -> None:
    for dtype in DTYPES:
        for window, sinks in ((1, 0), (1, 1), (5, 4), (16, 0), (33, 17), (64, 3), (100, 130), (500, 4), (2**40, 2**40)):
            for held, news, packed in (([400, 90, 33], [1, 1, 1], False), ([300, 77], [70, 70], False),
                                       ([350, 40, 129], [129, 1, 20], True)):
                s = step(held, news, heads=8, kv_heads=2, dtype=dtype, mx=mx, packed=packed, device=DEV, seed=window % 97)
                check(s, f"{dtype} {window} {sinks} {held}", window=window, sinks=sinks)


def test_long_contexts_are_split_and_joined() -> None:
    for dtype, mx in ((torch.bfloat16, False), (torch.float16, True), (torch.float32, False)):
        for held, news in (([9001], [1]), ([5003, 100, 1], [1, 1, 1]), ([6000], [9]), ([4100], [150])):
            s = step(held, news, heads=8, kv_heads=2, head_dim=128, dtype=dtype, mx=mx, page=64, device=DEV)
            check(s, f"{dtype} {held} {news}")
            check(s, f"{dtype} {held} {news} window", window=2500, sinks=7)


@pytest.fixture
def tuned():
    from ako_amd import _native

    def set_keys(items: int, keys: int) -> None:
        _native.set_tuning(3, 1, items)
        _native.set_tuning(3, 2, keys)

    yield set_keys
    set_keys(0, 0)


@pytest.mark.parametrize("items,keys", [(1, 1), (64, 64), (4096, 64), (65536, 1), (16, 65536)])
def test_however_the_keys_are_cut(tuned, items: int, keys: int) -> None:
    tuned(items, keys)
    for dtype, mx in ((torch.bfloat16, False), (torch.float16, True), (torch.float32, False)):
        for held, news, packed in (([900, 40, 1, 333], [1] * 4, False), ([700, 1000], [50, 50], False),
                                   ([600, 40, 1, 333, 0], [200, 1, 1, 90, 0], True)):
            s = step(held, news, heads=8, kv_heads=2, dtype=dtype, mx=mx, packed=packed, pad_rows=3 * packed, device=DEV)
            check(s, f"{dtype} {held} {news}")
            check(s, f"{dtype} {held} {news} window", window=100, sinks=40)


@pytest.mark.parametrize("packed", [False, True])
def test_many_sequences(packed: bool) -> None:
    """More sequences than a wavefront has lanes, empty ones among them."""
    for dtype in DTYPES:
        held = [(7 * i * i) % 300 if i % 9 else 0 for i in range(150)]
        held[70] = 2000
        news = [min(n, 1 + i % 5) for i, n in enumerate(held)] if packed else [3] * 150
        s = step(held, news, heads=4, kv_heads=2, dtype=dtype, packed=packed, pad_rows=70 * packed, device=DEV)
        check(s, str(dtype))
        if packed:  # and a few long ones: the many-row kernel
            s = step(held[60:140], [min(n, 40 * (i % 3)) for i, n in enumerate(held[60:140])], heads=4, kv_heads=2, dtype=dtype,
                     packed=True, device=DEV)
            check(s, f"{dtype} chunks")
        cos, sin = tables(2048, 64, DEV)
        before = [t.clone() for t in (s.k_pages, s.v_pages)]
        out = ako.rope_qk_paged(s.q, s.k, s.v, cos, sin, *s.where, **s.kw)
        if packed:
            check_write(s, out, cos, sin, "neox", before)


def test_a_wide_table_is_read_only_as_far_as_needed() -> None:
    s = step([50, 3], [1, 1], width=1 << 16, dtype=torch.float16, device=DEV)
    check(s)
    s = step([50, 63], [30, 30], width=1 << 16, dtype=torch.float16, device=DEV)
    check(s)


@pytest.mark.usefixtures("kernel")
@pytest.mark.parametrize("news", [1, 40])
def test_padding_and_short_sequences(news: int) -> None:
    for dtype in DTYPES:
        s = step([0, news - 1, news, news + 5, 2], [news] * 5, dtype=dtype, device=DEV)
        s.q[0] = math.nan  # rows that see nothing: what they hold does not matter
        out = attend(s)
        assert not out[0].any()
        check(s)
        e = step([], [], packed=True, pad_rows=news, dtype=dtype, device=DEV)
        assert not attend(e).any()


@pytest.mark.usefixtures("kernel")
@pytest.mark.parametrize("news", [1, 33])
def test_lengths_and_tables_that_make_no_sense(news: int) -> None:
    """Device-side indexes cannot be checked on the host: whatever they hold, nothing outside the
    tensors is touched, and sequences whose own indexes are right get right results."""
    s = step([60, 60, 60, 60, 60, 60], [news] * 6, page=8, dtype=torch.bfloat16, device=DEV)
    want, bound = attention64(s)
    s.lens[0], s.lens[1], s.lens[2] = -5, 2**31 - 1, 61 + 8 * 1000
    s.table[3], s.table[4] = 2**31 - 1, -2**31
    out = attend(s)
    assert not out[0].any() and not out[3].any() and not out[4].any()
    assert_within(out[5], want[5], bound[5])
    cos, sin = tables(64, 64, DEV)
    ako.rope_qk_paged(s.q, s.k, s.v, cos, sin, *s.where)
    ako.paged_read(*s.where, news)
    p = step([60, 60, 60], [news] * 3, page=8, packed=True, dtype=torch.bfloat16, device=DEV)
    for cu in ([0, 2**31 - 1, -7, 3], [-4, -3, -2, -1], [9, 6, 3, 0], [0, 0, 0, 10**6]):
        p.cu.copy_(torch.tensor(cu, dtype=torch.int64).int())
        ako.rope_qk_paged(p.q, p.k, p.v, cos, sin, *p.where, **p.kw)
        ako.paged_read(*p.where, p.rows, **p.kw)
        attend(p)
    torch.cuda.synchronize()


@pytest.mark.usefixtures("kernel")
@pytest.mark.parametrize("news", [1, 5, 40, 129])
@pytest.mark.parametrize("mx", [False, True])
def test_values_that_a_row_does_not_see_do_not_reach_it(mx: bool, news: int) -> None:
    for dtype in DTYPES:
        for poison in (math.nan,) if mx else (math.nan, math.inf, -math.inf):
            s = step([170, 200], [news, news], page=16, dtype=dtype, mx=mx, device=DEV, heads=8, kv_heads=2)
            bad = 0x7F if mx else poison
            def put(pages, i, j):
                raw = pages.view(torch.uint8) if mx else pages
                raw[s.table[i, j // 16], :, j % 16] = bad
            put(s.v_pages, 0, 170 - (news + 1) // 2)  # seen by the later half of the rows
            put(s.k_pages, 1, 200 - (news + 1) // 2)
            put(s.v_pages, 1, 10)  # before every row's window, behind the sinks
            put(s.k_pages, 0, 11)
            want, bound = attention64(s, window=20, sinks=2)
            out = attend(s, window=20, sinks=2)
            first = news - (news + 1) // 2  # rows before it
            assert torch.isfinite(out[:, :first]).all()
            assert_within(out[:, :first], want[:, :first], bound[:, :first], f"{dtype} {poison}")
            assert not torch.isfinite(out[:, first:]).all()


@pytest.mark.usefixtures("kernel")
@pytest.mark.parametrize("news", [1, 40])
def test_scores_of_minus_infinity(tuned, news: int) -> None:
    """Rows that see keys but nothing above -infinity are 0 / 0; one finite score is enough for a sum."""
    for dtype in DTYPES:
        for keys in (0, 64):
            tuned(0, keys)
            s = step([720, 90], [news, news], heads=8, kv_heads=2, page=16, dtype=dtype, device=DEV)
            s.k_pages[..., 0] = 1.0
            s.q[:, ::2, :, 0] = -math.inf
            want, bound = attention64(s)
            out = attend(s)
            assert out[:, ::2].isnan().all()
            assert_within(out, want, bound, f"{dtype} {keys}")
            s = step([720, 90], [news, news], heads=8, kv_heads=2, page=16, dtype=dtype, device=DEV)
            s.q[..., 0] = 1.0
            first = s.table[0, :37].long()
            s.table[0, :37] = -1
            want, bound = attention64(s)
            s.table[0, :37] = first.int()
            s.k_pages[first, ..., 0] = -math.inf  # a weight of 0, as if the keys were not there
            assert_within(attend(s), want, bound, f"{dtype} {keys} some")


@pytest.mark.parametrize("layout", ["heads", "tokens", "pair", "odd"])
def test_layouts(layout: str) -> None:
    for dtype, mx in ((torch.float16, False), (torch.bfloat16, True), (torch.float32, False), (torch.bfloat16, False)):
        for news in (1, 50):
            s = step([150, 70], [news, news], heads=8, kv_heads=2, head_dim=80, dtype=dtype, mx=mx, layout=layout,
                     fused=True, device=DEV)
            check(s, f"{dtype} {news}")


def test_scores_of_all_sizes() -> None:
    """Weights that are one, and scores whose exponentials would overflow or vanish without the maximum."""
    for dtype in DTYPES:
        for scale in (0.0, 1e-6, 1.0, 8.0, -0.5):
            for news in (1, 40):
                s = step([300, 64], [news, news], heads=4, kv_heads=2, dtype=dtype, device=DEV)
                check(s, f"{dtype} {scale}", scale=scale)


def test_ctypes_and_binding_agree() -> None:
    for mx in (False, True):
        s = step([60, 17], [9, 9], dtype=torch.float16, mx=mx, device=DEV)
        cos, sin = tables(64, 64, DEV)
        kw = (s.k_scales, s.v_scales, s.cu)
        a = ako.rope_qk_paged(s.q, s.k, s.v, cos, sin, *s.where, **s.kw)
        ka = [t.clone() for t in ako.paged_read(*s.where, 9, torch.float16, **s.kw)]
        b = paged_hip.rope_qk_paged_hip_ctypes(s.q, s.k, s.v, cos, sin, *s.where, "neox", *kw)
        kb = paged_hip.paged_read_hip_ctypes(*s.where, 9, torch.float16, *kw)
        assert torch.equal(a, b) and torch.equal(ka[0], kb[0]) and torch.equal(ka[1], kb[1])
        assert torch.equal(attend(s, window=30, sinks=2), paged_hip.paged_attention_hip_ctypes(s.q, *s.where, None, 30, 2, *kw))


@pytest.mark.parametrize("name,call,message", bad_calls(), ids=lambda x: x if isinstance(x, str) else "")
def test_refusals_of_both_bindings(name: str, call, message: str) -> None:
    from ako_amd import _native

    fast = _native.torch_binding()
    none = lambda s: (s.k_scales, s.v_scales, s.cu)  # noqa: E731
    tab = lambda cos: (cos.to(DEV),) * 2 if cos is not None else tables(64, 64, DEV)  # noqa: E731

    def fns(m, suffix):
        return (lambda s, style, cos: getattr(m, "rope_qk_paged" + suffix)(s.q, s.k, s.v, *tab(cos), *s.where, style, *none(s)),
                lambda s, rows, dtype: getattr(m, "paged_read" + suffix)(*s.where, rows, dtype, *none(s)),
                lambda s, o: getattr(m, "paged_attention" + suffix)(s.q, *s.where, o.get("scale"), o.get("window"),
                                                                   o.get("sinks", 0), *none(s)))

    said = []
    for f in (fns(fast, ""), fns(paged_hip, "_hip_ctypes")):
        s = step([9, 17], [1, 1], device=DEV)
        with pytest.raises(ValueError, match=message) as e:
            call(f, s)
        said.append(str(e.value))
    assert said[0] == said[1]


def test_other_streams() -> None:
    s = step([300, 77], [1, 1], dtype=torch.bfloat16, device=DEV)
    cos, sin = tables(512, 64, DEV)
    first = ako.rope_qk_paged(s.q, s.k, s.v, cos, sin, *s.where)
    want = attend(s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ako.rope_qk_paged(s.q, s.k, s.v, cos, sin, *s.where)
        got = attend(s)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, again) and torch.equal(want, got)


@pytest.mark.parametrize("mx", [False, True])
def test_captured_steps_follow_the_lengths(mx: bool) -> None:
    """Two graphs of the same step, replayed in turn with eager work between, as lengths grow."""
    s = step([200, 40, 0], [1, 1, 1], heads=8, kv_heads=2, dtype=torch.float16, mx=mx, device=DEV, spare=40, width=32)
    for i in range(3):  # room to grow
        free = [p for p in range(s.k_pages.shape[0]) if p not in set(s.table.flatten().tolist())]
        empty = (s.table[i] < 0).nonzero().flatten().tolist()[:4]
        s.table[i, empty] = torch.tensor(free[:len(empty)], dtype=torch.int32, device=DEV)
    cos, sin = tables(512, 64, DEV)

    def run():
        q = ako.rope_qk_paged(s.q, s.k, s.v, cos, sin, *s.where, **s.kw)
        return ako.paged_attention(q, *s.where, **s.kw), ako.paged_attention(q, *s.where, window=60, sinks=2, **s.kw)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run()
        graphs.append((g, out))
    for turn in range(6):
        s.lens += 1
        s.held = [n + 1 for n in s.held]
        s.q.copy_(torch.randn_like(s.q))
        s.k.copy_(torch.randn_like(s.k))
        g, out = graphs[turn % 2]
        g.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        want = run()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), turn
    s.q = ako.rope_qk_paged(s.q, s.k, s.v, cos, sin, *s.where, **s.kw)
    check(s)


def test_offsets_past_32_bits() -> None:
    """A pool of more than 2^31 elements, with the sequence's pages at its far end."""
    page, kvh, d = 64, 8, 128
    n = 2**31 // (page * kvh * d) + 40
    for dtype in (torch.float16, E4M3):
        k, v, ks, vs = ako.new_pages(n, kvh, page, d, dtype, device=DEV)
        g = torch.Generator(device=DEV).manual_seed(1)
        table = torch.tensor([[n - 1, 0, n - 2, n - 7]], dtype=torch.int32, device=DEV)
        lens = torch.zeros(1, dtype=torch.int32, device=DEV)
        cos, sin = tables(256, d, DEV)
        lens.fill_(230)
        q, kk, vv = (torch.randn(1, 230, h, d, generator=g, device=DEV).half() for h in (32, kvh, kvh))
        q = ako.rope_qk_paged(q, kk, vv, cos, sin, k, v, table, lens, k_scales=ks, v_scales=vs)
        s = step([230], [230], device=DEV)
        s.q, s.k_pages, s.v_pages, s.k_scales, s.v_scales, s.table, s.lens = q, k, v, ks, vs, table, lens
        check(s)
        got = ako.paged_read(*s.where, 230, torch.float16, **s.kw)
        for t, pages, codes in zip(got, (k, v), (ks, vs)):
            assert torch.equal(t[0].double(), stored(pages, codes, table, page, 0, 230)[0].half().double())
        assert torch.allclose(got[1][0].float(), vv[0].float(), rtol=2 ** -4 if ks is not None else 0, atol=0.01 * (ks is not None))
        del k, v, ks, vs, s, got
        torch.cuda.empty_cache()


def test_sequences_that_share_pages() -> None:
    s = step([80, 80], [1, 1], page=16, dtype=torch.bfloat16, device=DEV)
    s.table[1, :4] = s.table[0, :4]
    check(s)


@pytest.mark.usefixtures("kernel")
def test_results_do_not_change_from_run_to_run() -> None:
    s = step([3000, 900, 5], [7, 7, 7], heads=8, kv_heads=2, dtype=torch.bfloat16, device=DEV)
    first = attend(s)
    assert all(torch.equal(first, attend(s)) for _ in range(5))

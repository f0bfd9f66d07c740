"""The paged-cache entry points of the C ABI on a machine without a GPU: what they refuse, and that
the workspace that is asked for does for every window. A call that passes every check reaches the
launch and reports that there is no device (4)."""

from __future__ import annotations

import ctypes

import pytest
import torch
from hypothesis import given, settings
from hypothesis import strategies as st

from ako_amd import _native

pytestmark = pytest.mark.skipif(torch.cuda.is_available(),
                                reason="passes fake device addresses: runs only where no GPU is visible")

OK, INVALID, UNSUPPORTED, NO_DEVICE = 0, 1, 2, 4
F32, F16, BF16, E4M3 = 0, 1, 2, 3
MIB = 1 << 20
I3 = ctypes.c_int64 * 3
# One buffer each, far apart.
Q, K, V, COS, SIN, OUT, KP, VP, KS, VS, TABLE, LENS, CU, WS = ((i + 1) * (1 << 34) for i in range(14))


def dense(n0: int, n1: int, n2: int, d: int):
    return I3(n1 * n2 * d, n2 * d, d)


def cache(**kw) -> _native.PagedCache:
    a = dict(pages=8, kv_heads=2, page=16, d=64, n=2, width=4, tokens=2, dtype=F16, cu=None)
    a.update({k: v for k, v in kw.items() if k in a})
    mx = a["dtype"] == E4M3
    codes = -(-a["d"] // 32)
    st4 = dense(a["pages"], a["kv_heads"], a["page"], a["d"])
    sc4 = dense(a["pages"], a["kv_heads"], a["page"], codes) if mx else I3()
    c = _native.PagedCache(KP, VP, KS if mx else None, VS if mx else None, TABLE, LENS, a["cu"], st4, st4, sc4, sc4,
                           a["pages"], a["kv_heads"], a["page"], a["d"], a["n"], a["width"], a["width"], a["tokens"], a["dtype"])
    for k, v in kw.items():
        if k not in a:
            setattr(c, k, v)
    return c


def attention(c, heads=4, dtype=F16, scale=0.1, window=0, sinks=0, q=Q, out=OUT, ws=WS, size=None, strides=None):
    lib = _native.load()
    at = ctypes.addressof(c)
    need = lib.ako_paged_attention_workspace(at, heads, dtype)
    strides = strides or I3(heads * c.head_dim, heads * c.head_dim, c.head_dim)
    return lib.ako_paged_attention_fwd(q, strides, out, at, heads, scale, window, sinks, ws, max(need, 0) if size is None else size,
                                       dtype, None)


def write(c, heads=4, dtype=F16, tdt=F32, style=0, rows=64, st_row=None, q=Q, k=K, v=V, cos=COS, out=OUT):
    lib = _native.load()
    d, kvh = c.head_dim, c.kv_heads
    return lib.ako_rope_qk_paged_fwd(q, k, v, cos, SIN, out, ctypes.addressof(c), heads, I3(heads * d, heads * d, d),
                                     I3(kvh * d, kvh * d, d), I3(kvh * d, kvh * d, d), rows, d // 2 if st_row is None else st_row,
                                     dtype, tdt, style, None)


def read(c, dtype=F16, k=Q, v=OUT):
    return _native.load().ako_paged_read_fwd(ctypes.addressof(c), k, v, dtype, None)


def test_good_calls_reach_the_launch() -> None:
    for dtype in (F32, F16, BF16):
        for pages in (dtype, E4M3):
            for cu in (None, CU):
                c = cache(dtype=pages, cu=cu)
                assert attention(c, dtype=dtype) == write(c, dtype=dtype) == read(c, dtype=dtype) == NO_DEVICE


def test_empty_calls_are_done_at_once() -> None:
    c = cache(tokens=0)
    assert attention(c) == write(c) == read(c) == OK
    assert attention(cache(), heads=0) == OK


@pytest.mark.parametrize("status,change,message", [
    (UNSUPPORTED, dict(dtype=BF16), "pages of dtype"),
    (UNSUPPORTED, dict(dtype=9), "pages of dtype"),
    (UNSUPPORTED, dict(d=72), "head_dim"), (UNSUPPORTED, dict(d=272), "head_dim"), (UNSUPPORTED, dict(d=0), "head_dim"),
    (INVALID, dict(kv_heads=0), "at least 1"), (INVALID, dict(page=0), "at least 1"),
    (INVALID, dict(pages=-1), "negative"), (INVALID, dict(tokens=-1), "negative"), (INVALID, dict(n=-1), "negative"),
    (INVALID, dict(width=-1), "negative"),
    (INVALID, dict(width=1 << 27), "positions"), (INVALID, dict(page=1 << 31), "positions"),
    (INVALID, dict(tokens=1 << 31), "too many"), (INVALID, dict(n=1 << 31, tokens=1 << 31), "too many"),
    (INVALID, dict(tokens=3), "no multiple"), (INVALID, dict(n=0), "no multiple"),
    (INVALID, dict(table_stride=3), "rows overlap"),
    (INVALID, dict(k_pages=None), "null"), (INVALID, dict(seq_lens=None), "null"), (INVALID, dict(block_table=None), "null"),
    (INVALID, dict(k_scales=KS), "scales"), (INVALID, dict(dtype=E4M3, v_scales=None), "null"),
    (INVALID, dict(k_strides=I3(-1, 1, 1)), "negative"),
    (INVALID, dict(v_strides=I3(1 << 61, 1, 1)), "overflow"),
])
def test_caches_that_are_refused(status: int, change: dict, message: str) -> None:
    for call in (attention, write, read):
        assert call(cache(**change)) == status
        assert message in _native.last_error()
    assert _native.load().ako_paged_attention_workspace(ctypes.addressof(cache(**change)), 4, F16) in (-1, 0)


def test_attention_refusals() -> None:
    c = cache()
    for kw, message in ((dict(heads=3), "no multiple"), (dict(scale=float("nan")), "finite"), (dict(scale=float("inf")), "finite"),
                        (dict(window=-1), "window"), (dict(sinks=-1), "window"), (dict(q=None), "null"), (dict(out=None), "null"),
                        (dict(out=Q + 64), "overlaps"), (dict(out=KP + 64), "overlaps"), (dict(out=LENS), "overlaps"),
                        (dict(out=TABLE + 16), "overlaps"), (dict(strides=I3(-1, 1, 1)), "negative")):
        assert attention(c, **kw) == INVALID and message in _native.last_error(), kw
    assert attention(c, dtype=7) == UNSUPPORTED
    long = cache(pages=64, width=64)  # 1024 positions: key ranges may be split
    assert attention(long) == NO_DEVICE
    for kw in (dict(size=16), dict(ws=None), dict(ws=WS + 8)):
        assert attention(long, **kw) == INVALID and "workspace" in _native.last_error()
    for ws in (Q, OUT, KP, TABLE):
        assert attention(long, ws=ws) == INVALID and "overlaps" in _native.last_error()


def test_write_refusals() -> None:
    for kw, message in ((dict(k=None), "null"), (dict(cos=None), "null"), (dict(st_row=16), "row stride"), (dict(rows=-1), "negative"),
                        (dict(out=Q), "overlaps an input"), (dict(out=COS), "overlaps an input"), (dict(out=KP), "overlaps the cache"),
                        (dict(out=LENS), "overlaps the cache"), (dict(k=KP + 128), "pages overlap")):
        assert write(cache(), **kw) == INVALID and message in _native.last_error(), kw
    assert write(cache(), style=2) == UNSUPPORTED and write(cache(), tdt=5) == UNSUPPORTED
    d, page, kvh = 64, 16, 2
    row = kvh * page * d
    assert write(cache(v_pages=KP)) == INVALID and "rows of the cache" in _native.last_error()
    assert write(cache(k_strides=I3(row, page * d, 0))) == INVALID and "rows of the cache" in _native.last_error()
    assert write(cache(k_pages=LENS - 64)) == INVALID and "lengths" in _native.last_error()
    # Keys and values of a page in one block, and of a head: apart although their spans overlap.
    pair = dict(k_strides=I3(2 * row, page * d, d), v_strides=I3(2 * row, page * d, d))
    assert write(cache(v_pages=KP + 2 * row, **pair)) == NO_DEVICE
    assert write(cache(v_pages=KP + 2 * row - 32, **pair)) == INVALID
    tight = dict(k_strides=I3(2 * row, page * 2 * d, 2 * d), v_strides=I3(2 * row, page * 2 * d, 2 * d))
    assert write(cache(v_pages=KP + 2 * d, **tight)) == NO_DEVICE
    assert write(cache(dtype=E4M3, k_scales=KP)) == INVALID and write(cache(dtype=E4M3, k_scales=VS)) == INVALID


def test_tuning_keys() -> None:
    lib = _native.load()
    for key in (1, 2):
        assert lib.ako_set_tuning(3, key, 0) == OK and lib.ako_set_tuning(3, key, -1) == INVALID
        assert lib.ako_set_tuning(3, key, 65537) == INVALID
    assert lib.ako_set_tuning(3, 3, 2) == OK and lib.ako_set_tuning(3, 3, 0) == OK and lib.ako_set_tuning(3, 3, 3) == INVALID
    assert lib.ako_set_tuning(3, 4, 0) == INVALID and lib.ako_set_tuning(3, 0, 0) == INVALID


def test_read_refusals() -> None:
    assert read(cache(), k=None) == INVALID
    for kw in (dict(k=KP), dict(k=OUT), dict(v=LENS), dict(v=TABLE)):
        assert read(cache(), **kw) == INVALID and "overlaps" in _native.last_error()


@settings(max_examples=300, deadline=None)
@given(dtype=st.sampled_from([F32, F16, BF16]), mx=st.booleans(), heads=st.sampled_from([1, 2, 4, 8]), group=st.sampled_from([1, 2, 5, 8]),
       d=st.sampled_from([16, 64, 128, 256]), page=st.integers(1, 300), width=st.integers(0, 400), n=st.integers(1, 70),
       new=st.integers(1, 300), packed=st.booleans(), window=st.one_of(st.just(0), st.integers(1, 100000), st.just(2**40)),
       sinks=st.one_of(st.integers(0, 3000), st.just(2**40)), kernel=st.integers(0, 2))
def test_the_workspace_does_for_every_window(dtype, mx, heads, group, d, page, width, n, new, packed, window, sinks, kernel) -> None:
    _native.set_tuning(3, 3, kernel)
    try:
        workspace_does(dtype, mx, heads, group, d, page, width, n, new, packed, window, sinks)
    finally:
        _native.set_tuning(3, 3, 0)


def workspace_does(dtype, mx, heads, group, d, page, width, n, new, packed, window, sinks) -> None:
    c = cache(dtype=E4M3 if mx else dtype, kv_heads=heads, d=d, page=page, width=width, n=n, tokens=n * new,
              cu=CU if packed else None, pages=4)
    need = _native.load().ako_paged_attention_workspace(ctypes.addressof(c), heads * group, dtype)
    assert 0 <= need < 1 << 32
    assert attention(c, heads * group, dtype, window=window, sinks=sinks) == NO_DEVICE
    if need:
        assert attention(c, heads * group, dtype, size=need - 1) == INVALID

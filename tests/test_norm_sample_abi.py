"""The C entry points of the norms of q and k and of sampling on a machine without a GPU: what
they refuse. A call that passes every check reaches the launch and reports that there is no device (4)."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from ako_amd import _native
from tests.test_paged_abi import cache

pytestmark = pytest.mark.skipif(torch.cuda.is_available(),
                                reason="passes fake device addresses: runs only where no GPU is visible")

OK, INVALID, UNSUPPORTED, NO_DEVICE = 0, 1, 2, 4
F32, F16, BF16, E4M3 = 0, 1, 2, 3
I3 = ctypes.c_int64 * 3
NAN = math.nan
# One buffer each, far apart, and apart from those of a cache.
Q, K, V, QW, KW, COS, SIN, QO, KO, X, U, T, TK, TP, MP, OUT, WS = ((i + 32) * (1 << 34) for i in range(17))


def norm(batch=2, seq=3, heads=4, kv_heads=2, d=64, eps=1e-6, dtype=F16, wdt=F32, tdt=F32, style=0, st_row=None, q=Q, k=K, qw=QW,
         kw=KW, cos=COS, sin=SIN, qo=QO, ko=KO, qs=None, ks=None):
    qs = qs or I3(seq * heads * d, heads * d, d)
    ks = ks or I3(seq * kv_heads * d, kv_heads * d, d)
    return _native.load().ako_rmsnorm_rope_qk_fwd(q, k, qw, kw, cos, sin, qo, ko, batch, seq, heads, kv_heads, d, qs, ks,
                                                  d // 2 if st_row is None else st_row, eps, dtype, wdt, tdt, style, None)


def write(c=None, heads=4, eps=1e-6, dtype=F16, wdt=F32, tdt=F32, style=0, rows=64, q=Q, k=K, v=V, qw=QW, kw=KW, out=QO):
    c = c or cache()
    d, kvh = c.head_dim, c.kv_heads
    kv = I3(kvh * d, kvh * d, d)
    return _native.load().ako_rmsnorm_rope_qk_paged_fwd(q, k, v, qw, kw, COS, SIN, out, ctypes.addressof(c), heads,
                                                        I3(heads * d, heads * d, d), kv, kv, rows, d // 2, eps, dtype, wdt, tdt, style, None)


def draw(rows=4, vocab=1000, stride=None, dtype=F16, x=X, u=U, t=None, t1=1.0, tk=None, tk1=0, tp=None, tp1=1.0, mp=None, mp1=0.0,
         out=OUT, ws=WS, size=None):
    lib = _native.load()
    need = lib.ako_sample_workspace(rows, vocab, dtype)
    return lib.ako_sample_fwd(x, u, t, t1, tk, tk1, tp, tp1, mp, mp1, out, rows, vocab, vocab if stride is None else stride, ws,
                              max(need, 0) if size is None else size, dtype, None)


def test_good_calls_reach_the_launch() -> None:
    for dtype in (F32, F16, BF16):
        for weights in (dtype, F32):
            assert norm(dtype=dtype, wdt=weights) == norm(dtype=dtype, wdt=weights, style=1) == NO_DEVICE
            for pages in (dtype, E4M3):
                assert write(cache(dtype=pages), dtype=dtype, wdt=weights) == NO_DEVICE
        for vocab in (1, 1000, 131072, 1 << 22):
            assert draw(vocab=vocab, dtype=dtype) == draw(vocab=vocab, dtype=dtype, t=T, tk=TK, tp=TP, mp=MP) == NO_DEVICE
    assert norm(heads=0, q=None, qo=None, qw=None) == norm(kv_heads=0, k=None, ko=None, kw=None) == NO_DEVICE
    assert norm(d=2) == norm(d=512) == norm(eps=0.0) == norm(qs=I3(0, 0, 0), ks=I3(0, 0, 0)) == NO_DEVICE
    assert draw(stride=0) == draw(stride=5000) == draw(t1=0.0, tk1=5, tp1=0.0, mp1=1.0) == draw(t1=math.inf) == NO_DEVICE


def test_empty_calls_are_done_at_once() -> None:
    none = dict(q=None, k=None, qw=None, kw=None, cos=None, sin=None, qo=None, ko=None)
    assert norm(batch=0, **none) == norm(seq=0, **none) == norm(heads=0, kv_heads=0, **none) == OK
    assert write(cache(tokens=0)) == draw(rows=0, x=None, u=None, out=None, ws=None) == OK


@pytest.mark.parametrize("bad,code,words", [
    (dict(dtype=4), UNSUPPORTED, "dtype"), (dict(tdt=-1), UNSUPPORTED, "dtype"), (dict(style=2), UNSUPPORTED, "style"),
    (dict(wdt=BF16), UNSUPPORTED, "weight dtype"), (dict(wdt=7), UNSUPPORTED, "weight dtype"),
    (dict(eps=-1e-6), INVALID, "eps"), (dict(eps=NAN), INVALID, "eps"), (dict(batch=-1), INVALID, "negative size"),
    (dict(heads=-1), INVALID, "negative size"), (dict(d=63), UNSUPPORTED, "head_dim"), (dict(d=0), UNSUPPORTED, "head_dim"),
    (dict(d=514), UNSUPPORTED, "head_dim"), (dict(batch=1 << 20, seq=1 << 11), INVALID, "2\\^31"),
    (dict(heads=(1 << 23) + 1), INVALID, "2\\^23"), (dict(q=None), INVALID, "null"), (dict(kw=None), INVALID, "null"),
    (dict(cos=None), INVALID, "null"), (dict(ko=None), INVALID, "null"), (dict(st_row=31), INVALID, "table row stride"),
    (dict(qs=I3(0, -1, 64)), INVALID, "negative stride"), (dict(ks=I3(1 << 62, 64, 64)), INVALID, "address space"),
    (dict(qo=Q), INVALID, "overlaps"), (dict(ko=QO + 100), INVALID, "overlaps"), (dict(qo=KW), INVALID, "overlaps"), (dict(ko=SIN), INVALID, "overlaps"),
])
def test_norms_refuse(bad: dict, code: int, words: str) -> None:
    with pytest.raises(RuntimeError, match=words):
        assert norm(**bad) == code
        raise RuntimeError(_native.last_error())


@pytest.mark.parametrize("bad,code,words", [
    (dict(wdt=BF16), UNSUPPORTED, "weight dtype"), (dict(eps=NAN), INVALID, "eps"), (dict(qw=None), INVALID, "null"),
    (dict(kw=None), INVALID, "null"), (dict(k=None), INVALID, "null"), (dict(rows=-1), INVALID, "negative size"),
    (dict(style=3), UNSUPPORTED, "style"), (dict(tdt=9), UNSUPPORTED, "dtype"), (dict(out=QW), INVALID, "overlap"),
    (dict(out=Q), INVALID, "overlap"),
])
def test_norms_into_pages_refuse(bad: dict, code: int, words: str) -> None:
    with pytest.raises(RuntimeError, match=words):
        assert write(**bad) == code
        raise RuntimeError(_native.last_error())


@pytest.mark.parametrize("bad,code,words", [
    (dict(dtype=3), UNSUPPORTED, "dtype"), (dict(rows=-1), INVALID, "rows"), (dict(rows=1 << 31), INVALID, "rows"),
    (dict(vocab=0), INVALID, "vocab"), (dict(vocab=(1 << 22) + 1), INVALID, "vocab"), (dict(t1=-1.0), INVALID, "temperature"),
    (dict(t1=NAN), INVALID, "temperature"), (dict(tk1=-1), INVALID, "top_k"), (dict(tp1=1.5), INVALID, "top_p"),
    (dict(tp1=NAN), INVALID, "top_p"), (dict(mp1=-0.5), INVALID, "min_p"), (dict(x=None), INVALID, "null"),
    (dict(u=None), INVALID, "null"), (dict(out=None), INVALID, "null"), (dict(stride=-1), INVALID, "stride"),
    (dict(stride=1 << 62), INVALID, "address space"), (dict(out=X + 8), INVALID, "overlaps"), (dict(out=U), INVALID, "overlaps"),
    (dict(out=T, t=T), INVALID, "overlaps"), (dict(vocab=131072, ws=None), INVALID, "workspace"),
    (dict(vocab=131072, ws=WS + 4), INVALID, "workspace"), (dict(vocab=131072, size=1 << 10), INVALID, "workspace"),
    (dict(vocab=131072, ws=X), INVALID, "overlaps"), (dict(vocab=131072, ws=OUT), INVALID, "overlaps"),
    (dict(vocab=131072, ws=MP, mp=MP), INVALID, "overlaps"),
])
def test_sampling_refuses(bad: dict, code: int, words: str) -> None:
    with pytest.raises(RuntimeError, match=words):
        assert draw(**bad) == code
        raise RuntimeError(_native.last_error())


@pytest.mark.parametrize("sizes", [(-1, 100, F16), (1, 0, F16), (1 << 31, 5, F16), (1, (1 << 22) + 1, F16), (1, 100, 3)])
def test_the_workspace_is_refused_where_the_call_is(sizes) -> None:
    assert _native.load().ako_sample_workspace(*sizes) == -1 and "ako_sample_workspace" in _native.last_error()


def test_the_workspace_is_what_divided_rows_need() -> None:
    need = _native.load().ako_sample_workspace
    assert need(0, 131072, F32) == need(8, 1000, F32) == need(100000, 131072, F32) == 0
    one = need(1, 131072, F32)
    assert one > 0 and one % 16 == 0 and need(7, 131072, F32) == 7 * one

"""The paged-cache operations on a CPU: their plain form against the definitions in 64 bits,
what they refuse, and that the two host bindings refuse alike."""

from __future__ import annotations

import math

import pytest
import torch

import ako_amd as ako
from ako_amd import _native
from ako_amd.ops import paged_hip
from ako_amd.ops.paged_ref import dequantize_rows, quantize_rows
from ako_amd.ops.rope_ref import rope_ref
from tests._paged import E4M3, Step, assert_within, attention64, e4m3_64, places, step, stored, tables

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_matches_64_bits(dtype, mx: bool) -> None:
    for held, news, packed in (([33, 1, 17], [1, 1, 1], False), ([40, 5, 0, 21], [7, 5, 0, 3], True),
                               ([20, 9], [4, 4], False)):
        s = step(held, news, dtype=dtype, mx=mx, packed=packed, pad_rows=2 if packed else 0, head_dim=48, page=7)
        for opts in ({}, {"window": 6}, {"window": 3, "sinks": 5}, {"scale": 0.3}):
            want, bound = attention64(s, **opts)
            assert_within(ako.paged_attention(s.q, *s.where, **opts, **s.kw), want, bound, f"{held} {opts}")


def test_rows_that_see_nothing_are_zero() -> None:
    s = step([0, 3, 5], [4, 4, 4], dtype=torch.float32)  # the first two have fewer positions than rows
    out = ako.paged_attention(s.q, *s.where)
    assert not out[0].any() and not out[1, 0].any() and out[1, 1:].any() and torch.isfinite(out).all()
    want, bound = attention64(s)
    assert_within(out, want, bound)


def test_absent_pages_are_not_seen() -> None:
    s = step([40, 40], [1, 1], page=8)
    s.table[0, 1] = -1
    s.table[1, :] = 10 ** 6
    want, bound = attention64(s)
    out = ako.paged_attention(s.q, *s.where)
    assert_within(out, want, bound)
    assert not out[1].any()


def test_values_that_a_row_does_not_see_do_not_reach_it() -> None:
    s = step([12], [4], page=4)
    j = 10  # seen by the last two rows only
    s.v_pages[s.table[0, j // 4], :, j % 4] = math.nan
    s.k_pages[s.table[0, 11 // 4], :, 11 % 4] = math.inf
    want, bound = attention64(s)
    out = ako.paged_attention(s.q, *s.where)
    assert torch.isfinite(out[0, :2]).all() and out[0, 2:].isnan().all()
    assert_within(out[:, :2], want[:, :2], bound[:, :2])


def test_quantised_rows_follow_the_format() -> None:
    g = torch.Generator().manual_seed(3)
    for d in (16, 32, 48, 80, 128):
        x = torch.randn(50, 3, d, generator=g) * torch.exp2(torch.randint(-30, 30, (50, 3, 1), generator=g).float())
        x[0], x[1, 0, 3], x[2, 1, 5], x[3, 2] = 0.0, math.inf, math.nan, 448.0
        x[4, 0, 0], x[5] = 448.0 * (1 + 2 ** -23), 1e-40
        q, codes = quantize_rows(x)
        values, want = e4m3_64(x.double())
        assert torch.equal(codes.double(), want)
        got = dequantize_rows(q, codes, torch.float32).double()
        assert torch.equal(got.isnan(), values.isnan()) and torch.equal(got.nan_to_num(), values.nan_to_num())
        fine = x.isfinite().double() * x.double().nan_to_num(0, 0, 0).abs()
        unit = torch.exp2(want - 127).repeat_interleave(32, -1)[..., :d]
        assert ((got - x.double()).abs().nan_to_num() <= torch.maximum(fine * 2 ** -4, unit * 2.0 ** -10)).all()


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("style", ["neox", "interleaved"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_write_then_read(dtype, style: str, mx: bool) -> None:
    for held, news, packed in (([9, 30], [1, 1], False), ([12, 3, 0, 25], [5, 3, 0, 9], True)):
        s = step(held, news, dtype=dtype, mx=mx, packed=packed, pad_rows=packed * 2, page=7, head_dim=48)
        cos, sin = tables(64, 48)
        before = [t.clone() for t in (s.k_pages, s.v_pages)]
        out = ako.rope_qk_paged(s.q, s.k, s.v, cos, sin, *s.where, style, **s.kw)
        check_write(s, out, cos, sin, style, before)


def check_write(s: Step, out, cos, sin, style, before) -> None:
    """q, the pages and what is read back, against the rotation in the rows' type (bit for bit) and
    the format in 64 bits; slots that the step does not write keep their bytes."""
    at = places(s)
    flat = [x.flatten(0, -3) for x in (s.q, s.k, s.v)]
    mx = s.k_scales is not None
    o = out.flatten(0, -3)
    pad = set(range(o.shape[0])) - {t for t, _, _ in at}
    assert not o[list(pad)].any()
    rows = torch.tensor([t for t, _, _ in at], device=o.device)
    pos = torch.tensor([p for _, _, p in at], device=o.device)
    turned = [rope_ref(x[rows][None], cos[pos], sin[pos], style)[0] for x in flat[:2]]
    assert torch.equal(o[rows], turned[0])
    page = s.k_pages.shape[2]
    kr, vr = ako.paged_read(*s.where, s.rows, s.q.dtype, **s.kw)
    assert not kr.flatten(0, -3)[list(pad)].any() and not vr.flatten(0, -3)[list(pad)].any()
    kr, vr = kr.flatten(0, -3)[rows], vr.flatten(0, -3)[rows]
    if mx:
        wide = rope_ref(flat[1][rows].float()[None], cos[pos].float(), sin[pos].float(), style)[0].double()
        assert torch.equal(kr, e4m3_64(wide)[0].to(s.q.dtype)) and torch.equal(vr, e4m3_64(flat[2][rows].double())[0].to(s.q.dtype))
    else:
        assert torch.equal(kr, turned[1]) and torch.equal(vr, flat[2][rows])
    raw = lambda t: t.view(torch.uint8) if t.dtype == E4M3 else t.view(torch.int32 if t.dtype == torch.float32 else torch.int16)  # noqa: E731
    written = torch.zeros(s.k_pages.shape[0], page, dtype=torch.bool, device=o.device)
    for _, i, p in at:
        written[s.table[i, p // page], p % page] = True
    kept = ~written[:, None, :, None].expand(s.k_pages.shape)
    for now, was in zip((s.k_pages, s.v_pages), before):
        assert torch.equal(raw(now)[kept], raw(was)[kept])


def test_positions_without_a_slot() -> None:
    s = step([20, 6, 9], [1, 1, 1], page=4)
    s.table[2, 2] = -1  # position 8
    cos, sin = tables(18, 64)  # position 19 has no table row
    before = [s.k_pages.clone(), s.v_pages.clone()]
    out = ako.rope_qk_paged(s.q, s.k, s.v, cos, sin, *s.where)
    assert out[0].isnan().all() and out[2].isnan().all() and torch.isfinite(out[1]).all()
    changed = (s.k_pages.nan_to_num(7) != before[0].nan_to_num(7)).any(-1).any(1).nonzero().tolist()
    assert changed == [[int(s.table[1, 1]), 1]]


def test_read_of_whole_sequences() -> None:
    s = step([10, 0, 23, 5], [10, 0, 23, 5], packed=True, pad_rows=3, mx=True, page=4, dtype=torch.bfloat16)
    k, v = ako.paged_read(*s.where, s.q.shape[0], torch.float16, **s.kw)
    want = torch.cat([stored(s.k_pages, s.k_scales, s.table, 4, i, n)[0] for i, n in enumerate(s.held)])
    assert k.dtype == torch.float16 and torch.equal(k[:38].double(), want.half().double()) and not k[38:].any()
    assert v.shape == (41, 2, 64)


def test_empty_calls() -> None:
    s = step([0], [0])
    assert ako.paged_attention(s.q, *s.where).shape == s.q.shape == (1, 0, 4, 64)
    assert ako.paged_read(*s.where, 0)[0].shape == (1, 0, 2, 64)
    e = step([], [], packed=True, pad_rows=2)
    assert not ako.paged_attention(e.q, *e.where, **e.kw).any()
    cos, sin = tables(4, 64)
    assert not ako.rope_qk_paged(e.q, e.k, e.v, cos, sin, *e.where, **e.kw).any()


def bad_calls():
    """(name, call, message): every refusal, for a call of rope_qk_paged, paged_read and paged_attention."""
    def attention(**change):
        opts = {k: change.pop(k) for k in ("scale", "window", "sinks") if k in change}
        def call(fns, s):
            for k, f in change.items():
                setattr(s, k, f(getattr(s, k)) if callable(f) else f)
            return fns[2](s, opts)
        return call

    def write(style="neox", cos=None, **change):
        def call(fns, s):
            for k, f in change.items():
                setattr(s, k, f(getattr(s, k)) if callable(f) else f)
            return fns[0](s, style, cos)
        return call

    def read(rows=1, dtype=None):
        return lambda fns, s: fns[1](s, rows, dtype)

    return [
        ("pages differ", attention(v_pages=lambda t: t[..., :32]), "alike"),
        ("head size", attention(k_pages=lambda t: t[..., :24], v_pages=lambda t: t[..., :24]), "multiple of 16"),
        ("page type", attention(k_pages=lambda t: t.double(), v_pages=lambda t: t.double()), "pages must be"),
        ("page rows", attention(k_pages=lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)), "contiguous in head_dim"),
        ("scales not wanted", attention(k_scales=torch.ones(1)), "are for float8"),
        ("scales missing", attention(k_pages=lambda t: t.to(E4M3), v_pages=lambda t: t.to(E4M3)), "need k_scales"),
        ("table type", attention(table=lambda t: t.long()), "2-D int32"),
        ("table rows", attention(table=lambda t: t.repeat(1, 2)[:, ::2] if t.shape[1] > 1 else t.repeat(1, 4)[:, ::2]), "rows must be contiguous"),
        ("table width", attention(table=lambda t: t[:, :1].expand(-1, 2 ** 27)), "contiguous|names more"),
        ("lengths", attention(lens=lambda t: t[:1]), "seq_lens must be"),
        ("lengths type", attention(lens=lambda t: t.long()), "seq_lens must be"),
        ("cu", attention(cu=torch.zeros(2, dtype=torch.int32)), "cu_seqlens must be"),
        ("rows", attention(q=lambda t: t[0]), "q must be"),
        ("row size", attention(q=lambda t: t[..., :32]), "does not match the pages"),
        ("sequences", attention(q=lambda t: t[:1]), "sequences"),
        ("row type", attention(q=lambda t: t.double()), "q must be float32"),
        ("types differ", attention(q=lambda t: t.half()), "the pages"),
        ("groups", attention(q=lambda t: t[:, :, :3]), "no multiple"),
        ("scale", attention(scale=math.inf), "scale must be finite"),
        ("window", attention(window=0), "window must be"),
        ("sinks", attention(window=4, sinks=-1), "window must be"),
        ("style", write(style="other"), "Unknown RoPE style"),
        ("k heads", write(k=lambda t: t[:, :, :1]), "k .* does not match the pages"),
        ("v rows", write(v=lambda t: t.repeat(1, 2, 1, 1)), "v .* does not match q"),
        ("v type", write(v=lambda t: t.half()), "v is torch.float16"),
        ("tables", write(cos=torch.ones(8, 16)), "tables must be"),
        ("read rows", read(rows=-1), "rows must be"),
        ("read type", read(dtype=torch.float64), "dtype must be"),
        ("read other type", read(dtype=torch.float16), "dtype is"),
    ]


PUBLIC = (
    lambda s, style, cos: ako.rope_qk_paged(s.q, s.k, s.v, *((cos, cos) if cos is not None else tables(64, 64)), *s.where, style, **s.kw),
    lambda s, rows, dtype: ako.paged_read(*s.where, rows, dtype, **s.kw),
    lambda s, opts: ako.paged_attention(s.q, *s.where, **opts, **s.kw),
)


@pytest.mark.parametrize("name,call,message", bad_calls(), ids=lambda x: x if isinstance(x, str) else "")
def test_refusals(name: str, call, message: str) -> None:
    with pytest.raises(ValueError, match=message):
        call(PUBLIC, step([9, 17], [1, 1]))


def test_hip_path_refuses_cpu_tensors() -> None:
    s = step([9, 17], [1, 1])
    cos, sin = tables(32, 64)
    fast = _native.torch_binding()
    assert fast is not None
    none = (None, None, None)
    for a, b in ((lambda: fast.paged_attention(s.q, *s.where, None, None, 0, *none),
                  lambda: paged_hip.paged_attention_hip_ctypes(s.q, *s.where)),
                 (lambda: fast.paged_read(*s.where, 1, None, *none), lambda: paged_hip.paged_read_hip_ctypes(*s.where, 1)),
                 (lambda: fast.rope_qk_paged(s.q, s.k, s.v, cos, sin, *s.where, "neox", *none),
                  lambda: paged_hip.rope_qk_paged_hip_ctypes(s.q, s.k, s.v, cos, sin, *s.where))):
        with pytest.raises(ValueError, match="GPU tensor") as x:
            a()
        with pytest.raises(ValueError, match="GPU tensor") as y:
            b()
        assert str(x.value) == str(y.value)

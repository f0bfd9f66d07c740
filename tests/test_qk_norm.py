"""RMSNorm of the heads of q and k with RoPE in the same pass, dense and into the pages of a cache,
against the formulas in 64 bits; refusals; strides, types, other streams, captured calls."""

from __future__ import annotations

import math

import pytest
import torch

import ako_amd as ako
from ako_amd import _native
from ako_amd.ops import paged_hip, qk_norm
from tests._paged import E4M3, U32, assert_within, e4m3_64, places, step, tables

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
EPS = 1e-6


def turned64(x, weight, cos, sin, eps, style):
    """``(value, error)`` of normed and rotated heads in 64 bits: x (..., rows, heads, d), tables (rows, d / 2).

    In 32 bits the sum of squares is off by at most d / 2 + 7 roundings of itself (chains of up
    to 16 and a tree, or a library's order), which the square root halves; mean, eps, root,
    both products, the rotation's products and its sum add at most 12. Together
    (d / 2 + 16) roundings of |a c| + |b n|.
    """
    d = x.shape[-1]
    x = x.double()
    y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / d + eps) * weight.double()
    c, n = cos.double()[:, None], sin.double()[:, None]
    a, b = (y[..., : d // 2], y[..., d // 2:]) if style == "neox" else (y[..., 0::2], y[..., 1::2])
    parts = (a * c - b * n, a * n + b * c), ((a * c).abs() + (b * n).abs(), (a * n).abs() + (b * c).abs())
    value, size = (torch.cat(p, -1) if style == "neox" else torch.stack(p, -1).flatten(-2) for p in parts)
    return value, size * (U32 * (d / 2 + 16))


def rounded(value, error, dtype):
    """How far a result of ``dtype`` may be from ``value``: the error, and half a step of the type."""
    f = torch.finfo(dtype)
    return error + (f.eps / 2 if dtype != torch.float32 else U32) * (value.abs() + error) + f.smallest_normal * f.eps


def inputs(batch, seq, heads, kv_heads, d, dtype, device, seed=0, fused=False, wdtype=None):
    g = torch.Generator().manual_seed(seed)
    scale = torch.exp2(torch.randint(-3, 4, (batch, seq, heads + kv_heads, 1), generator=g).float())
    row = (torch.randn(batch, seq, heads + kv_heads, d, generator=g) * scale).to(dtype).to(device)
    q, k = row[:, :, :heads], row[:, :, heads:]
    if not fused:
        q, k = q.contiguous(), k.contiguous()
    qw, kw = ((1 + 0.3 * torch.randn(d, generator=g)).to(wdtype or dtype).to(device) for _ in range(2))
    return q, k, qw, kw


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("style", ["neox", "interleaved"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_head_size(dtype, style: str, device: str) -> None:
    sizes = list(range(2, 68, 2)) + [72, 80, 96, 112, 126, 128, 136, 160, 192, 254, 256, 258, 320, 510, 512]
    for i, d in enumerate(sizes):
        q, k, qw, kw = inputs(2, 3, (4, 3, 1)[i % 3], (2, 3, 1)[i % 3], d, dtype, device, i, fused=i % 2 == 1,
                              wdtype=(None, torch.float32)[i % 2])
        cos, sin = tables(3, d, device, (torch.float32, dtype)[i % 2])
        out = ako.rmsnorm_rope_qk(q, k, qw, kw, cos, sin, EPS, style)
        for x, w, y in ((q, qw, out[0]), (k, kw, out[1])):
            assert y.shape == x.shape and y.dtype == dtype and y.is_contiguous()
            want, error = turned64(x, w, cos, sin, EPS, style)
            assert_within(y, want, rounded(want, error, dtype), f"{d}")


@pytest.mark.parametrize("device", DEVICES)
def test_strides_weights_and_eps(device: str) -> None:
    q, k, qw, kw = inputs(3, 5, 4, 2, 64, torch.bfloat16, device, 1)
    cos, sin = tables(9, 64, device)
    cases = {
        "heads first": (q.transpose(1, 2).contiguous().transpose(1, 2), k.transpose(1, 2).contiguous().transpose(1, 2)),
        "batches expanded": (q[:1].expand(3, -1, -1, -1), k[:1].expand(3, -1, -1, -1)),
        "every other element": (q.repeat_interleave(2, -1)[..., ::2], k.repeat_interleave(2, -1)[..., ::2]),
        "odd start": tuple(torch.cat([x.flatten(), x.flatten()[:3]]).roll(3)[3:].view(x.shape) for x in (q, k)),
    }
    for name, (a, b) in cases.items():
        for eps in (0.0, 1e-6, 1.0):
            for w in ((qw, kw), (qw.double(), kw), (qw.repeat_interleave(2)[::2], kw.float())):
                out = ako.rmsnorm_rope_qk(a, b, *w, cos[2:7], sin[2:7], eps)
                for x, v, y in ((a, w[0], out[0]), (b, w[1], out[1])):
                    want, error = turned64(x, v, cos[2:7], sin[2:7], eps, "neox")
                    assert_within(y, want, rounded(want, error, x.dtype), name)


@pytest.mark.parametrize("device", DEVICES)
def test_zero_infinite_and_missing_rows(device: str) -> None:
    q, k, qw, kw = inputs(1, 6, 2, 1, 32, torch.float16, device, 2)
    q[0, 0, 0], q[0, 1, 0, 3], q[0, 2, 1, 7], q[0, 3, 0] = 0.0, math.inf, math.nan, 65504.0
    q[0, 4, 1] = 2.0 ** -24
    cos, sin = tables(6, 32, device)
    out, _ = ako.rmsnorm_rope_qk(q, k, qw, kw, cos, sin, EPS)
    assert not out[0, 0, 0].any() and out[0, 2, 1].isnan().all()
    bad = out[0, 1, 0].isnan()  # inf * 0, and its partner; the others are 0
    assert bad.nonzero().flatten().tolist() == [3, 19] and not out[0, 1, 0][~bad].any()
    for row, head in ((3, 0), (4, 1), (5, 0), (1, 1)):
        want, error = turned64(q[0, row:row + 1, head:head + 1], qw, cos[row:row + 1], sin[row:row + 1], EPS, "neox")
        assert_within(out[0, row:row + 1, head:head + 1], want, rounded(want, error, torch.float16))
    # No heads on one side, no tokens, no batch.
    assert ako.rmsnorm_rope_qk(q[:, :, :0], k, qw, kw, cos, sin)[0].shape == (1, 6, 0, 32)
    a, b = ako.rmsnorm_rope_qk(q[:, :, :0], k, qw, kw, cos, sin)
    assert torch.equal(b, ako.rmsnorm_rope_qk(q, k, qw, kw, cos, sin)[1])
    a, b = ako.rmsnorm_rope_qk(q, k[:, :, :0], qw, kw, cos, sin)
    assert torch.equal(a[0, 5], out[0, 5]) and b.numel() == 0
    assert ako.rmsnorm_rope_qk(q[:, :0], k[:, :0], qw, kw, cos[:0], sin[:0])[1].shape == (1, 0, 1, 32)
    assert ako.rmsnorm_rope_qk(q[:0], k[:0], qw, kw, cos, sin)[0].shape == (0, 6, 2, 32)


def check_paged(s, out, qw, kw, cos, sin, style, before) -> None:
    """A normed write against 64 bits; the slots that the step does not write keep their bytes."""
    at = places(s)
    rows = torch.tensor([t for t, _, _ in at], device=out.device)
    pos = torch.tensor([p for _, _, p in at], device=out.device)
    o, dtype = out.flatten(0, -3), s.q.dtype
    pad = sorted(set(range(o.shape[0])) - set(rows.tolist()))
    assert not o[pad].any()
    want, error = turned64(s.q.flatten(0, -3)[rows], qw, cos[pos], sin[pos], EPS, style)
    assert_within(o[rows], want, rounded(want, error, dtype), "q")
    kr, vr = (x.flatten(0, -3)[rows] for x in ako.paged_read(*s.where, s.rows, torch.float32 if s.k_scales is not None else dtype, **s.kw))
    v = s.v.flatten(0, -3)[rows]
    want, error = turned64(s.k.flatten(0, -3)[rows], kw, cos[pos], sin[pos], EPS, style)
    if s.k_scales is None:
        assert_within(kr, want, rounded(want, error, dtype), "k")
        assert torch.equal(vr, v)
    else:
        # A value within its error of a rounding border may go either way, and so may a block's
        # scale: one step of e4m3, 2^-3 of the value or 2^-9 of the scale that the largest may have.
        held, codes = e4m3_64(want)
        unit = torch.exp2(codes + 1 - 127).repeat_interleave(32, -1)[..., : want.shape[-1]]
        near = torch.zeros_like(want, dtype=torch.bool)
        for side in (want - error, want + error):
            near |= e4m3_64(side)[0] != held
        near = torch.nn.functional.pad(near, (0, -near.shape[-1] % 32)).unflatten(-1, (-1, 32))
        shifted = (e4m3_64(want * (1 + 2 ** -16))[1] != codes) | (e4m3_64(want * (1 - 2 ** -16))[1] != codes)
        either = (near | shifted[..., None]).flatten(-2)[..., : want.shape[-1]]
        step8 = torch.where(either, torch.maximum(held.abs() * 2 ** -3, unit * 2.0 ** -9), torch.zeros_like(held))
        assert_within(kr, held, step8, "k, 8 bits")
        assert torch.equal(vr.double(), e4m3_64(v.double())[0])
        assert either.double().mean() < 0.02
    taken = torch.zeros(s.k_pages.shape[0], s.k_pages.shape[2], dtype=torch.bool, device=out.device)
    for _, i, p in at:
        taken[s.table[i, p // s.k_pages.shape[2]].long(), p % s.k_pages.shape[2]] = True
    for pages, old in zip((s.k_pages, s.v_pages), before):
        raw = lambda t: t.transpose(1, 2)[~taken].contiguous().view(torch.uint8)  # noqa: E731
        assert torch.equal(raw(pages), raw(old))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("style", ["neox", "interleaved"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_into_pages(dtype, style: str, mx: bool, device: str) -> None:
    for i, d in enumerate([16, 32, 48, 64, 80, 96, 112, 128, 160, 192, 240, 256]):
        heads, kv_heads = ((4, 2), (3, 3), (7, 1))[i % 3]
        for held, news, packed in (([9, 30], [1, 1], False), ([12, 3, 0, 25, 70], [5, 3, 0, 9, 64], True), ([40, 33], [33, 33], False)):
            s = step(held, news, heads=heads, kv_heads=kv_heads, head_dim=d, dtype=dtype, mx=mx, packed=packed,
                     pad_rows=3 * packed, page=(1, 7, 16)[i % 3], device=device, seed=i,
                     layout=("heads", "tokens", "pair", "odd")[i % 4], fused=i % 2 == 1, q_scale=8.0)
            cos, sin = tables(80, d, device, (torch.float32, dtype)[i % 2])
            _, _, qw, kw = inputs(1, 1, 1, 1, d, dtype, device, i, wdtype=(None, torch.float32)[i % 2])
            before = [t.clone() for t in (s.k_pages, s.v_pages)]
            out = ako.rope_qk_paged(s.q, s.k, s.v, cos, sin, *s.where, style, q_weight=qw, k_weight=kw, eps=EPS, **s.kw)
            check_paged(s, out, qw, kw, cos, sin, style, before)


@pytest.mark.parametrize("device", DEVICES)
def test_positions_without_a_slot(device: str) -> None:
    s = step([20, 6, 9], [1, 1, 1], page=4, device=device)
    s.table[2, 2] = -1
    cos, sin = tables(18, 64, device)
    w = torch.ones(64, device=device)
    before = s.k_pages.clone()
    out = ako.rope_qk_paged(s.q, s.k, s.v, cos, sin, *s.where, q_weight=w, k_weight=w)
    assert out[0].isnan().all() and out[2].isnan().all() and torch.isfinite(out[1]).all()
    changed = (s.k_pages.nan_to_num(7) != before.nan_to_num(7)).any(-1).any(1).nonzero().tolist()
    assert changed == [[int(s.table[1, 1]), 1]]


# ------------------------------------------------------------------------- refusals --
def bad_dense():
    w = torch.ones(64)
    cos = torch.ones(3, 32)
    good = dict(q=torch.ones(2, 3, 4, 64), k=torch.ones(2, 3, 2, 64), q_weight=w, k_weight=w, cos=cos, sin=cos, eps=EPS, style="neox")
    change = [
        (dict(style="other"), "RoPE style"), (dict(q=good["q"][0]), "Expected x of shape"), (dict(cos=cos[:2], sin=cos[:2]), "cos/sin"),
        (dict(k=good["k"][:1]), "must match"), (dict(k=good["k"].half()), "must match"),
        (dict(q=good["q"].double(), k=good["k"].double()), "float32/float16/bfloat16"),
        (dict(q_weight=w[:32]), "q_weight of shape"), (dict(k_weight=w[None]), "k_weight of shape"),
        (dict(eps=-1.0), "eps must be"), (dict(eps=math.nan), "eps must be"),
        (dict(q=torch.ones(1, 3, 1, 514), k=torch.ones(1, 3, 1, 514), cos=torch.ones(3, 257), sin=torch.ones(3, 257)), "head_dim must be"),
        (dict(q=torch.ones(1, 3, 1, 7), k=torch.ones(1, 3, 1, 7)), "must be even"),
    ]
    return [({**good, **c}, message) for c, message in change]


@pytest.mark.parametrize("kw,message", bad_dense(), ids=[m for _, m in bad_dense()])
def test_dense_refusals(kw, message: str) -> None:
    with pytest.raises(ValueError, match=message):
        ako.rmsnorm_rope_qk(**kw)


def bad_norms():
    w = torch.ones(64)
    return [((None, w, EPS), "both be given"), ((w, None, EPS), "both be given"), ((w[:32], w, EPS), "q_weight of shape"),
            ((w, w[:, None], EPS), "k_weight of shape"), ((w, w, -1e-6), "eps must be"), ((w, w, math.nan), "eps must be")]


@pytest.mark.parametrize("args,message", bad_norms())
def test_paged_refusals(args, message: str) -> None:
    s = step([5, 9], [1, 1])
    qw, kw, eps = args
    before = s.k_pages.clone()
    with pytest.raises(ValueError, match=message):
        ako.rope_qk_paged(s.q, s.k, s.v, *tables(16, 64), *s.where, q_weight=qw, k_weight=kw, eps=eps)
    assert torch.equal(s.k_pages.nan_to_num(7), before.nan_to_num(7))


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")
def test_both_bindings_refuse_alike_and_launch_alike() -> None:
    fast = _native.torch_binding()
    assert fast is not None
    for kw, message in bad_dense():
        kw = {k: v.cuda() if torch.is_tensor(v) else v for k, v in kw.items()}
        said = []
        for fn in (fast.rmsnorm_rope_qk, qk_norm.rmsnorm_rope_qk_hip_ctypes):
            with pytest.raises(ValueError, match=message) as e:
                fn(**kw)
            said.append(str(e.value))
        assert said[0] == said[1]
    for (qw, kw, eps), message in bad_norms():
        s = step([5, 9], [1, 1], device="cuda")
        qw, kw = (None if t is None else t.cuda() for t in (qw, kw))
        said = []
        for fn in (fast.rope_qk_paged, paged_hip.rope_qk_paged_hip_ctypes):
            with pytest.raises(ValueError, match=message) as e:
                fn(s.q, s.k, s.v, *tables(16, 64, "cuda"), *s.where, "neox", None, None, None, qw, kw, eps)
            said.append(str(e.value))
        assert said[0] == said[1]
    args = (*inputs(2, 5, 4, 2, 80, torch.float16, "cuda"), *tables(5, 80, "cuda"))
    for a, b in zip(fast.rmsnorm_rope_qk(*args, EPS, "neox"), qk_norm.rmsnorm_rope_qk_hip_ctypes(*args, EPS, "neox")):
        assert torch.equal(a, b)
    w = torch.rand(64, device="cuda")
    outs = []
    for fn in (fast.rope_qk_paged, paged_hip.rope_qk_paged_hip_ctypes):
        s = step([5, 9], [3, 3], device="cuda", mx=True, dtype=torch.bfloat16)
        o = fn(s.q, s.k, s.v, *tables(16, 64, "cuda"), *s.where, "neox", s.k_scales, s.v_scales, None, w, w, EPS)
        outs.append((o, s.k_pages.view(torch.uint8), s.k_scales))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


# ------------------------------------------------------------------ large, streams, graphs --
@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")
def test_many_tokens_and_a_side_stream() -> None:
    q, k, qw, kw = inputs(3, 1111, 32, 8, 128, torch.bfloat16, "cpu", 5, fused=True)
    cos, sin = tables(1111, 128, "cuda")
    q, k, qw, kw = (t.cuda() for t in (q, k, qw, kw))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = ako.rmsnorm_rope_qk(q, k, qw, kw, cos, sin, EPS)
    torch.cuda.current_stream().wait_stream(side)
    for x, w, y in ((q, qw, out[0]), (k, kw, out[1])):
        want, error = turned64(x, w, cos, sin, EPS, "neox")
        assert_within(y, want, rounded(want, error, x.dtype))


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")
def test_captured_steps_follow_the_lengths() -> None:
    s = step([9, 14], [1, 1], page=4, dtype=torch.float16, device="cuda", width=8)
    s.table.copy_(torch.arange(16, device="cuda").view(2, 8) % s.k_pages.shape[0])
    pool = torch.zeros(16, *s.k_pages.shape[1:], dtype=torch.float16, device="cuda")
    s.table.copy_(torch.arange(16, device="cuda").view(2, 8))
    s.k_pages, s.v_pages = pool, pool.clone()
    cos, sin = tables(32, 64, "cuda")
    qw, kw = (torch.rand(64, device="cuda") + 0.5 for _ in range(2))
    run = lambda: ako.rope_qk_paged(s.q, s.k, s.v, cos, sin, *s.where, q_weight=qw, k_weight=kw, eps=EPS)  # noqa: E731
    run()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    for turn in range(4):
        s.lens.add_(1)
        s.q.copy_(torch.randn_like(s.q))
        s.k.copy_(torch.randn_like(s.k))
        g.replay()
        got, pages = out.clone(), s.k_pages.clone()
        torch.cuda.synchronize()
        s.held = s.lens.tolist()
        s.k_pages.zero_()
        assert torch.equal(run(), got)
        at = places(s)
        for _, i, p in at:
            page, slot = int(s.table[i, p // 4]), p % 4
            assert torch.equal(s.k_pages[page, :, slot], pages[page, :, slot])
        s.k_pages.copy_(pages)


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")
@pytest.mark.parametrize("which", range(4))
def test_gradients_that_are_not_formed_are_told_of(which: int) -> None:
    """The results are the same and carry no gradient; nothing is said where none can be expected."""
    import warnings

    args = [*inputs(1, 3, 2, 1, 32, torch.float32, "cuda"), *tables(3, 32, "cuda")]
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        want = ako.rmsnorm_rope_qk(*args)
        args[which] = args[which].detach().requires_grad_()
        with torch.no_grad():
            ako.rmsnorm_rope_qk(*args)
    with pytest.warns(UserWarning, match="no backward pass"):
        got = ako.rmsnorm_rope_qk(*args)
    for a, b in zip(got, want):
        assert torch.equal(a, b) and not a.requires_grad


def test_gradients_on_a_cpu_are_the_formulas() -> None:
    import warnings

    args = [*inputs(1, 2, 2, 1, 8, torch.float32, "cpu"), *tables(2, 8)]
    args[:4] = [t.double().requires_grad_() for t in args[:4]]

    def turned(q, k, qw, kw):
        out = []
        for x, w in ((q, qw), (k, kw)):
            y = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w
            a, b = y.chunk(2, -1)
            c, n = (t.double()[:, None] for t in args[4:])
            out.append(torch.cat((a * c - b * n, a * n + b * c), -1))
        return out

    seeds = [torch.randn(t.shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64) for i, t in enumerate(args[:2])]
    want = torch.autograd.grad(turned(*args[:4]), args[:4], seeds)
    low = [t.detach().float().requires_grad_() for t in args[:4]]
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        got = torch.autograd.grad(ako.rmsnorm_rope_qk(*low, *args[4:]), low, [s.float() for s in seeds])
    for a, b in zip(got, want):
        # Sums of at most 16 products of four 32-bit factors, each of some size around 1: 16 * 8 half steps.
        assert (a.double() - b).abs().max() <= 128 * 2.0 ** -24 * max(1.0, b.abs().max().item())

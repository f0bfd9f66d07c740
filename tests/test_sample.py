"""Drawing tokens: against the definition in 64 bits, one row at a time; ties, ruled-out tokens,
infinities, extreme settings, refusals, other streams, captured calls."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import ako_amd as ako
from ako_amd import _native
from ako_amd.ops.sample import sample_hip_ctypes

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def f32(v) -> float:
    return float(np.float32(v))


def allowed(x: np.ndarray, u: float, t: float, k: int, p: float, low: float) -> set[int]:
    """The tokens that may come out for one row, from the definition in 64 bits: one, unless a
    sum comes closer to a border than the kernel's weights are fine, V 2^-(S+1) of the largest for a sum of
    V of them, where S = min(51, 62 - log2 V rounded up); then also the token behind that border."""
    v = x.size
    slack = v * 2.0 ** -(min(51, 62 - math.ceil(math.log2(max(v, 2)))) + 1) + 1e-13
    live = np.flatnonzero(x > -math.inf)
    if not live.size:
        return {-1}
    order = live[np.argsort(-x[live], kind="stable")]
    if not t > 0:
        return {int(order[0])}
    top = x[order[0]]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.exp((x[order] - top) / t)
    w = np.where(x[order] == top, 1.0, np.nan_to_num(w))
    order, w = order[w > 2.0 ** -60], w[w > 2.0 ** -60]
    if k > 0:
        order, w = order[:k], w[:k]
    before = np.cumsum(w) - w
    lengths = {order.size}
    if p < 1:
        want = max(p, 0.0) * w.sum()
        lengths = {max(1, int((before < want + d).sum())) for d in (-slack, 0.0, slack)}
    out = set()
    for n in lengths:
        o, ww = order[:n], w[:n]
        if low > 0:
            keep = ww >= min(low, 1.0)
            o, ww = o[keep], ww[keep]
        by = np.argsort(o)
        o, upto = o[by], np.cumsum(ww[by])
        target = (u if u > 0 else 0.0) * upto[-1]
        for d in (-slack, 0.0, slack):
            out.add(int(o[min(int((upto <= target + d).sum()), o.size - 1)]))
    return out


def check(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, settled=0.99) -> torch.Tensor:
    """Every row's token is one that may come out, and all but few rows have only one such."""
    got = ako.sample(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    assert got.dtype == torch.int64 and got.shape == (logits.shape[0],) and got.device == logits.device
    x, uu, one = logits.double().cpu().numpy(), u.cpu().numpy(), 0
    row = lambda v, r: v[r].item() if torch.is_tensor(v) else v if isinstance(v, int) else f32(v)  # noqa: E731
    for r in range(logits.shape[0]):
        may = allowed(x[r], float(uu[r]), row(temperature, r), row(top_k, r), row(top_p, r), row(min_p, r))
        assert int(got[r]) in may, (r, int(got[r]), may, [row(v, r) for v in (temperature, top_k, top_p, min_p)])
        one += len(may) == 1
    assert one >= settled * logits.shape[0]
    return got


def rows(n, v, dtype, device, seed=0, scale=3.0, masked=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, v, generator=g) * scale
    if masked:
        x.masked_fill_(torch.rand(n, v, generator=g) < 0.7, -math.inf)
    return x.to(dtype).to(device), torch.rand(n, generator=g).to(device)


SETTINGS = [{}, dict(temperature=0.7), dict(top_k=1), dict(top_k=7), dict(top_k=400), dict(top_p=0.9), dict(top_p=0.3),
            dict(min_p=0.05), dict(top_k=50, top_p=0.8), dict(top_k=50, top_p=0.8, min_p=0.1, temperature=1.5),
            dict(top_p=0.95, min_p=0.01, temperature=2.0), dict(temperature=0.0), dict(temperature=0.0, top_p=0.1)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_setting(dtype, device: str) -> None:
    for i, kw in enumerate(SETTINGS):
        for masked in (False, True):
            check(*rows(12, 1000 + i, dtype, device, i, masked=masked), **kw)


@pytest.mark.parametrize("device", DEVICES)
def test_every_width(device: str) -> None:
    for v in (1, 2, 3, 7, 8, 9, 63, 64, 65, 127, 129, 1023, 1025, 2047, 2049, 4095, 4097, 8191, 8193, 20000, 32768, 32771):
        for kw in ({}, dict(top_k=5), dict(top_p=0.7)):
            check(*rows(5, v, DTYPES[v % 3], device, v), **kw)


@pytest.mark.parametrize("device", DEVICES)
def test_draws_follow_the_weights(device: str) -> None:
    """Uniform numbers in the middle of every token's share give every token, in order."""
    x = torch.tensor([0.3, -math.inf, 2.0, 2.0, math.nan, -1.0, 1.5], device=device)
    w = torch.exp(x.double()).nan_to_num(0.0)
    upto = w.cumsum(0) / w.sum()
    mid = (upto - w / w.sum() / 2)[[0, 2, 3, 5, 6]].float()
    assert ako.sample(x.expand(5, -1), mid).tolist() == [0, 2, 3, 5, 6]
    assert ako.sample(x.expand(4, -1), torch.tensor([0.0, 0.25, 0.75, 1 - 2.0 ** -24], device=device), top_k=2).tolist() == [2, 2, 3, 3]


@pytest.mark.parametrize("device", DEVICES)
def test_ties_go_to_the_lowest_index(device: str) -> None:
    for v in (10, 5000, 70000):  # more equal ones than the kernel holds in its list
        x = torch.zeros(4, v, device=device)
        x[1, v // 2] = 1.0
        x[2], x[2, ::3] = -1.0, 0.0
        u = torch.tensor([0.999, 0.9999, 0.9999, 0.5], device=device)
        k = v // 5
        assert ako.sample(x, u, top_k=k)[0].item() == int(0.999 * k)
        assert ako.sample(x, u, temperature=0.0).tolist() == [0, v // 2, 0, 0]
        assert ako.sample(x, u, top_k=1).tolist() == [0, v // 2, 0, 0]
        check(x, u, top_k=k, settled=0.5)
        check(x, u, top_p=0.4, settled=0.5)
        check(x, u, top_k=2 * k, top_p=0.6, settled=0.5)
        check(-x.to(torch.bfloat16), u, top_k=3 * k, min_p=0.5, settled=0.5)


@pytest.mark.parametrize("device", DEVICES)
def test_rows_that_rule_everything_or_much_out(device: str) -> None:
    inf = math.inf
    x = torch.tensor([[-inf] * 5, [math.nan] * 5, [-inf, math.nan, 3.0, -inf, -inf], [inf, 1.0, inf, -inf, math.nan],
                      [-3e38, -3.4e38, -inf, -3e38, -3e38], [3.4e38, -3.4e38, 0.0, 3.4e38, 1.0], [0.0, -0.0, 0.0, -0.0, -inf]],
                     device=device)
    u = torch.full((7,), 0.6, device=device)
    for kw in ({}, dict(top_k=3), dict(top_p=0.9), dict(min_p=0.1), dict(temperature=inf), dict(temperature=1e-30),
               dict(temperature=inf, top_k=2, top_p=0.9)):
        got = ako.sample(x, u, **kw).tolist()
        assert got[:3] == [-1, -1, 2] and got[3] == 2 and got[5] == 3, kw
        check(x, u, **kw)
    assert ako.sample(x, u, temperature=0.0).tolist() == [-1, -1, 2, 0, 0, 0, 0]
    assert ako.sample(x, u, top_k=2).tolist()[6] == 1 and ako.sample(x, u).tolist()[6] == 2


@pytest.mark.parametrize("device", DEVICES)
def test_extreme_settings(device: str) -> None:
    x, u = rows(30, 3000, torch.float32, device, 3)
    for t in (1e-4, 0.01, 10.0, 1000.0, 1e30, math.inf):
        for kw in ({}, dict(top_k=100), dict(top_p=0.5), dict(top_k=2000, top_p=0.9, min_p=0.3)):
            # At high temperatures all weights are nearly 1 and top_p times their sum nearly a whole
            # number, 0.5 * 3000 or 0.9 * 2000: every row's sum stops at a border.
            check(x, u, temperature=t, settled=0.9 if t <= 10 else 0.0, **kw)
    assert torch.equal(ako.sample(x, u, top_p=0.0), ako.sample(x, u, temperature=0.0))
    assert torch.equal(ako.sample(x, u, min_p=1.0), ako.sample(x, u, temperature=0.0))
    assert torch.equal(ako.sample(x, u, top_k=10 ** 9), ako.sample(x, u))
    assert torch.equal(ako.sample(x, u, top_p=1.0, min_p=0.0, top_k=3000), ako.sample(x, u))


@pytest.mark.parametrize("device", DEVICES)
def test_settings_and_numbers_per_row(device: str) -> None:
    x, u = rows(64, 2500, torch.float32, device, 4)
    g = torch.Generator().manual_seed(1)
    pick = lambda values, dtype: torch.tensor(values, dtype=dtype)[torch.randint(0, len(values), (64,), generator=g)].to(device)  # noqa: E731
    t, k = pick([0.0, -1.0, 0.5, 1.0, 2.0], torch.float32), pick([0, -5, 1, 9, 300, 2 ** 31 - 1], torch.int32)
    p, m = pick([-0.5, 0.0, 0.3, 0.9, 1.0, 1.5], torch.float32), pick([-1.0, 0.0, 0.1, 1.0, 7.0], torch.float32)
    got = check(x, u, t, k, p, m)
    for r in (0, 13, 40):  # alone as in the batch
        one = slice(r, r + 1)
        assert int(ako.sample(x[one], u[one], temperature=t[one], top_k=k[one], top_p=p[one], min_p=m[one])) == int(got[r])
    t[:8], p[8:16], m[16:24] = math.nan, math.nan, math.nan
    got = ako.sample(x, u, temperature=t, top_k=k, top_p=p, min_p=m)
    want = ako.sample(x, u, temperature=t.nan_to_num(0.0), top_k=k, top_p=p.nan_to_num(1.0), min_p=m.nan_to_num(0.0))
    assert torch.equal(got, want)
    odd = torch.tensor([-1.0, math.nan, 0.0, 1.0, 2.0, math.inf], device=device)
    got = ako.sample(x[:1].expand(6, -1), odd, top_k=10).tolist()
    assert got[0] == got[1] == got[2] and got[3] == got[4] == got[5]
    best = x[0].topk(10).indices
    assert got[0] == int(best.min()) and got[3] == int(best.max())


@pytest.mark.parametrize("device", DEVICES)
def test_strides_and_empty_batches(device: str) -> None:
    x, u = rows(6, 700, torch.float16, device, 5)
    want = ako.sample(x, u, top_k=20)
    wide = torch.full((6, 2, 703), 9.0, dtype=torch.float16, device=device)
    wide[:, 1, 3:] = x
    for y in (wide[:, 1, 3:], x.t().contiguous().t(), x.repeat_interleave(2, -1)[:, ::2]):
        assert torch.equal(ako.sample(y, u, top_k=20), want)
    assert ako.sample(x[:0], u[:0]).shape == (0,)


# ------------------------------------------------------------------------- refusals --
def bad():
    x, u = torch.zeros(3, 10), torch.zeros(3)
    good = dict(logits=x, uniform=u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    change = [(dict(logits=x[0]), "rows, vocab"), (dict(logits=x.double()), "float32/float16"), (dict(logits=x[:, :0]), "vocab must be"),
              (dict(uniform=u[:2]), "uniform must be"), (dict(uniform=u.double()), "uniform must be"),
              (dict(uniform=torch.zeros(6)[::2]), "uniform must be"),
              (dict(temperature=-1.0), "temperature must be at least 0, got -1.0"), (dict(temperature=math.nan), "temperature must be"),
              (dict(temperature=u.half()), "temperature must be a number or"), (dict(top_k=u), "top_k must be a number or"),
              (dict(top_k=-1), "top_k must be a whole"), (dict(top_k=1.5), "top_k must be a whole"), (dict(top_p=1.5), "top_p must be 0 to 1"),
              (dict(top_p=-0.1), "top_p must be 0 to 1"), (dict(top_p=math.nan), "top_p must be 0 to 1"), (dict(min_p=2), "min_p must be 0 to 1"),
              (dict(min_p=u[:1]), "min_p must be a number or"), (dict(top_p=u[:, None]), "top_p must be a number or")]
    return [({**good, **c}, m) for c, m in change]


@pytest.mark.parametrize("kw,message", bad(), ids=lambda x: x if isinstance(x, str) else "")
def test_refusals(kw, message: str) -> None:
    x, u = kw.pop("logits"), kw.pop("uniform")
    with pytest.raises(ValueError, match=message):
        ako.sample(x, u, **kw)


def test_a_vocabulary_past_the_limit_is_refused() -> None:
    with pytest.raises(ValueError, match="vocab must be"):
        ako.sample(torch.zeros(1, 1).expand(1, 2 ** 22 + 1), torch.zeros(1))


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")
def test_both_bindings_alike() -> None:
    fast = _native.torch_binding()
    for kw, message in bad():
        there = lambda t: t.cuda() if t.is_contiguous() else t.repeat_interleave(2).cuda()[::2]  # noqa: E731
        kw = {k: there(v) if torch.is_tensor(v) else v for k, v in kw.items()}
        said = []
        for fn in (fast.sample, sample_hip_ctypes):
            with pytest.raises(ValueError, match=message) as e:
                fn(**kw)
            said.append(str(e.value))
        assert said[0] == said[1]
    x, u = rows(9, 5000, torch.bfloat16, "cuda", 6)
    k = torch.arange(9, dtype=torch.int32, device="cuda")
    for kw in (dict(temperature=0.8, top_k=k, top_p=0.9, min_p=0.0), dict(temperature=u + 0.5, top_k=40, top_p=u, min_p=u / 10)):
        assert torch.equal(fast.sample(x, u, **kw), sample_hip_ctypes(x, u, **kw))


# ----------------------------------------------------------------- sizes, streams, graphs --
@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")
@pytest.mark.parametrize("vocab", [65536, 131073, 262144, 1000003, 2 ** 22])
def test_large_vocabularies(vocab: int) -> None:
    for i, kw in enumerate(({}, dict(top_k=50, top_p=0.9), dict(top_k=30000), dict(top_p=0.9), dict(top_p=0.5, temperature=0.6),
                            dict(min_p=0.02, top_p=0.99, temperature=1.5))):
        check(*rows(3, vocab, DTYPES[i % 3], "cuda", i, scale=(2.0, 4.0)[i % 2], masked=i % 3 == 1), settled=0.0, **kw)


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")
def test_the_cpu_form_agrees() -> None:
    x, u = rows(40, 32000, torch.float32, "cpu", 8)
    for kw in SETTINGS:
        assert torch.equal(ako.sample(x, u, **kw), ako.sample(x.cuda(), u.cuda(), **kw).cpu()), kw


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")
def test_streams_and_captured_calls() -> None:
    x, u = rows(20, 32000, torch.float16, "cuda", 9)
    t, k = torch.rand(20, device="cuda") + 0.5, torch.randint(0, 60, (20,), device="cuda", dtype=torch.int32)
    run = lambda: ako.sample(x, u, temperature=t, top_k=k, top_p=0.9)  # noqa: E731
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
        u.copy_(torch.rand(20, device="cuda"))
        x.copy_(torch.randn(20, 32000, device="cuda") * (turn + 1))
        t.copy_(torch.rand(20, device="cuda"))
        k.copy_(torch.randint(0, 6000, (20,), device="cuda", dtype=torch.int32))
        want = run()
        g, out = graphs[turn % 2]
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_the_token_does_not_depend_on_the_division(dtype) -> None:
    """Rows of 40000 tokens are divided over workgroups up to 78 of them at once, and whole from 79 on."""
    gen = torch.Generator("cuda").manual_seed(3)
    x = (torch.randn(79, 40000, generator=gen, device="cuda") * 3).to(dtype)
    x[::5] = x[::5].round()  # many equal ones
    x[3, 1:] = -math.inf
    x[4] = math.nan
    x[5] = 1.5  # more alike than a list holds
    u = torch.rand(79, generator=gen, device="cuda")
    for kw in ({}, dict(temperature=0.0), dict(top_k=50), dict(top_k=5000), dict(top_p=0.9), dict(top_k=1000, top_p=0.5), dict(min_p=0.02),
               dict(temperature=torch.linspace(0, 2, 79, device="cuda"), top_p=torch.linspace(0, 1, 79, device="cuda"),
                    top_k=torch.arange(79, dtype=torch.int32, device="cuda") * 40)):
        whole = ako.sample(x, u, **kw)
        part = {k: v[:78] if torch.is_tensor(v) else v for k, v in kw.items()}
        assert torch.equal(ako.sample(x[:78], u[:78], **part), whole[:78]), kw
        one = {k: v[7:8] if torch.is_tensor(v) else v for k, v in kw.items()}
        assert torch.equal(ako.sample(x[7:8], u[7:8], **one), whole[7:8]), kw
        assert whole[4] == -1 and whole[3] == 0


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,vocab", [(torch.float16, 24577), (torch.float16, 24601), (torch.bfloat16, 32001), (torch.bfloat16, 32767),
                                         (torch.float32, 12289), (torch.float32, 12301), (torch.float32, 16383)])
def test_rows_of_four_rounds_and_a_rest(dtype, vocab: int, device: str) -> None:
    """Kept in LDS with more than three rounds of packets and elements behind the last whole one."""
    for kw in ({}, dict(top_k=5), dict(top_k=5000), dict(top_p=0.7), dict(top_k=6000, top_p=0.8), dict(min_p=0.01)):
        check(*rows(5, vocab, dtype, device, vocab), **kw)


@pytest.mark.parametrize("device", DEVICES)
def test_numbers_that_float32_does_not_hold(device: str) -> None:
    """They are rounded to it: past its largest to infinity, next to 0 and 1 to those."""
    x, u = rows(6, 500, torch.float32, device, 12)
    assert torch.equal(ako.sample(x, u, temperature=1e39), ako.sample(x, u, temperature=math.inf))
    assert torch.equal(ako.sample(x, u, temperature=1e-50), ako.sample(x, u, temperature=0.0))
    assert torch.equal(ako.sample(x, u, top_p=1 - 1e-12, min_p=1e-60), ako.sample(x, u))
    assert torch.equal(ako.sample(x, u, top_k=10 ** 30), ako.sample(x, u))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_signalling_nan_is_ruled_out_too(dtype, device: str) -> None:
    """NaN of either sign whose first mantissa bit is clear, in rows in LDS, whole in memory and divided."""
    bits, quiet = {torch.float32: (torch.int32, 0x400000), torch.float16: (torch.int16, 0x200), torch.bfloat16: (torch.int16, 0x40)}[dtype]
    inf = torch.tensor([math.inf, -math.inf], dtype=dtype).view(bits)
    for n, v in ((6, 50), (6, 5000), (6, 70000), (100, 33000)):
        x, u = rows(n, v, dtype, "cpu", v)
        raw, clean = x.clone().view(bits), x.clone()
        for k in range(2):
            at = torch.randint(0, v, (v // 7,), generator=torch.Generator().manual_seed(k))
            raw[:, at], clean[:, at] = inf[k] + 1, -math.inf
        raw[4], clean[4] = inf[0] + 1, -math.inf
        raw[5], clean[5] = inf[1] + quiet - 1, -math.inf
        raw[5, 3], clean[5, 3] = x.view(bits)[5, 3], x[5, 3]
        y = raw.view(dtype).to(device)
        assert torch.equal(y.cpu().view(bits), raw)
        for kw in ({}, dict(temperature=0.0), dict(top_k=7), dict(top_p=0.5), dict(top_k=30, top_p=0.9, min_p=0.01)):
            got = ako.sample(y, u.to(device), **kw)
            assert torch.equal(got, ako.sample(clean.to(device), u.to(device), **kw)) and got[4:6].tolist() == [-1, 3]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_min_p_of_one_keeps_the_largest_alone(dtype, device: str) -> None:
    """Also of logits so close that their weights are 1 in 64 bits."""
    least = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    x = torch.arange(40, dtype=torch.float64).mul(least).to(dtype).flip(0).roll(7).expand(5, -1).contiguous().to(device)
    x[:, 20] = x[:, 7]  # and one more like the largest
    u = torch.tensor([0.0, 0.3, 0.499, 0.501, 0.999], device=device)
    for kw in (dict(min_p=1.0), dict(min_p=torch.ones(5, device=device)), dict(min_p=1.0, top_p=0.9), dict(min_p=1.0, temperature=30.0)):
        assert ako.sample(x, u, **kw).tolist() == [7, 7, 7, 20, 20]

"""The paged key/value cache and the attention that reads it, as measurable cases.

A serving program keeps the keys and values of its sequences in pages of a
pool, ``(pages, kv_heads, page_size, head_dim)``, and finds them through a
block table. Three operators work on it:

* write      RoPE of a step's queries and keys, with the rotated keys and the
             values stored at the sequences' next positions, in the model's
             type or as e4m3 with one power-of-two scale per 32 elements;
* read       the stored keys and values of given positions, as dense rows;
* attention  of a step's tokens over all that their sequences hold, causal,
             with grouped heads and, if asked, a sliding window beside a few
             first tokens that stay visible.

``listed()`` gives the fixed cases, ``draw`` one more from the ranges they
stand for, ``prepare`` what a program holds before the call, ``run`` one pass
(``own`` false: elementary torch operations; true: the library's operators),
``work`` the bytes and operations a pass cannot do without and ``exact`` its
results in 64 bits.

Ranges (``draw``): 1-64 sequences, one new token or up to 2048 each (all alike,
or packed one after the other), up to 65536 positions, 4-32 query heads in
groups of 1-8, head sizes of 64-256, pages of 16-256 positions and odd ones,
float16 / bfloat16 / float32, pages in that type or in e4m3.
"""

from __future__ import annotations

import math
import random

import torch

#: Whether ``run`` calls the library's operators or computes their plain form.
own = False

DEVICE = "cuda"
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
ROPE_BASE = 10000.0
#: Positions per sequence, values gathered per tensor, scores and operations of
#: the largest listed case of each; no drawn case has more.
MAX_LEN = 65536
MAX_CACHE = 16 * 65536 * 8 * 128
MAX_SCORES = 2048 * 32 * 32768
MAX_TOKENS = 8192


# --------------------------------------------------------------------- cases --
def write_case(batch, new, max_len, heads, kv_heads, head_dim, page, dtype, *, mx, style="neox", ragged=False):
    return {"kind": "write", "batch": batch, "new": new, "max_len": max_len, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "dtype": dtype, "mx": mx, "style": style, "ragged": ragged,
            "window": 0, "sinks": 0}


def read_case(batch, max_len, kv_heads, head_dim, page, dtype, *, mx, ragged=False):
    return {"kind": "read", "batch": batch, "new": max_len, "max_len": max_len, "heads": kv_heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "dtype": dtype, "mx": mx, "ragged": ragged,
            "window": 0, "sinks": 0}


def attention_case(batch, new, max_len, heads, kv_heads, head_dim, page, dtype, *, mx=False, ragged=False,
                   window=0, sinks=0):
    return {"kind": "attention", "batch": batch, "new": new, "max_len": max_len, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "dtype": dtype, "mx": mx, "ragged": ragged,
            "window": window, "sinks": sinks}


def listed() -> list[dict]:
    return [
        # A serving batch's decode step: rotate and store one token each.
        {"name": "write_step", **write_case(64, 1, 640, 32, 8, 128, 64, "float16", mx=False)},
        # Prompts stored in 8 bits, and what was stored read back.
        {"name": "write_prompts_mx8", **write_case(4, 2048, 2048, 32, 8, 128, 64, "bfloat16", mx=True)},
        # The whole 8-bit cache of a ragged batch unpacked, as for moving it to another process.
        {"name": "read_batch_mx8", **read_case(16, 4096, 8, 128, 16, "bfloat16", mx=True, ragged=True)},
        # One short sequence's cache as dense rows: pages of an odd size.
        {"name": "read_one", **read_case(1, 513, 4, 64, 7, "float32", mx=False)},
        # The last of 128 greedy steps after a prompt of 512, one sequence: the smallest call, all latency.
        {"name": "step_one", **attention_case(1, 1, 640, 32, 32, 128, 64, "float16")},
        # A serving batch's decode step over contexts of all lengths, grouped heads, small pages.
        {"name": "step_batch", **attention_case(64, 1, 8192, 32, 8, 128, 16, "bfloat16", ragged=True)},
        # Long contexts in 8 bits, one token each: nothing but cache bytes.
        {"name": "step_long_mx8", **attention_case(16, 1, 65536, 32, 8, 128, 64, "bfloat16", mx=True)},
        # A decode step with a sliding window and 4 first tokens that stay visible.
        {"name": "step_window", **attention_case(32, 1, 32768, 32, 8, 128, 32, "float16", window=4096, sinks=4)},
        # A prompt of 512, one sequence: causal attention of a prompt pass.
        {"name": "prompt", **attention_case(1, 512, 512, 32, 32, 128, 64, "float16")},
        # A chunk of 2048 tokens at the end of a context of 32768: the largest call.
        {"name": "chunk_long", **attention_case(1, 2048, 32768, 32, 8, 128, 64, "bfloat16")},
        # Chunks of prompts and single tokens packed in one step, windowed, 8-bit pages, heads of 80.
        {"name": "mixed_mx8", **attention_case(16, 300, 4097, 32, 8, 80, 16, "bfloat16", mx=True, ragged=True,
                                               window=1024, sinks=16)},
        # Full precision, heads of 64 in groups of 8, odd lengths.
        {"name": "chunk_f32", **attention_case(2, 257, 1025, 32, 4, 64, 64, "float32")},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    while True:
        kind = rng.choice(["write", "read", "attention", "attention", "attention"])
        dtype = rng.choice(["float16", "bfloat16", "bfloat16", "float32"])
        kv_heads, group = rng.choice([4, 4, 8, 8, 32]), rng.choice([1, 4, 8, 8])
        head_dim, page = rng.choice([64, 80, 128, 128, 256]), rng.choice([16, 16, 32, 64, 64, 256, 7, 24])
        heads = min(32, kv_heads * group)
        batch, ragged, mx = _log_int(rng, 1, 64), rng.random() < 0.5, rng.random() < 0.5
        if kind == "write":
            new = rng.choice([1, _log_int(rng, 2, 2048)])
            case = write_case(batch, new, new + _log_int(rng, 1, 4096), heads, kv_heads, head_dim, page, dtype,
                              mx=mx, style=rng.choice(["neox", "neox", "interleaved"]), ragged=ragged)
            if batch * new > MAX_TOKENS:
                continue
        elif kind == "read":
            case = read_case(batch, _log_int(rng, 16, 8192), kv_heads, head_dim, page, dtype, mx=mx, ragged=ragged)
            if batch * case["max_len"] > 8 * MAX_TOKENS:
                continue
        else:
            new = rng.choice([1, 1, _log_int(rng, 2, 2048)])
            window = rng.choice([0, 0, _log_int(rng, 16, 8192)])
            case = attention_case(batch, new, new + _log_int(rng, 1, MAX_LEN - new), heads, kv_heads, head_dim, page,
                                  dtype, mx=mx, ragged=ragged, window=window, sinks=rng.choice([0, 4, 33]) if window else 0)
            if batch * new * heads * case["max_len"] > MAX_SCORES or batch * new > MAX_TOKENS:
                continue
        if batch * case["max_len"] * kv_heads * head_dim <= MAX_CACHE:
            return case


def lengths(case) -> tuple[list[int], list[int]]:
    """Positions held by each sequence after the step, and new tokens of each: the same for every seed."""
    n, new, top = case["batch"], case["new"], case["max_len"]
    rng = random.Random(n * 1000003 + new * 1009 + top)
    if not case["ragged"]:  # new tokens alike; contexts within an eighth of the longest
        return [top - (rng.randrange(max(1, (top - new) // 8 + 1)) if i else 0) for i in range(n)], [new] * n
    if case["kind"] == "read":
        lens = [_log_int(rng, 1, top) if i else top for i in range(n)]
        return lens, lens
    news = [new if not i else 1 if rng.random() < 0.6 else _log_int(rng, 1, new) for i in range(n)]
    return [top if not i else m + _log_int(rng, 1, top - m) for i, m in enumerate(news)], news


# ------------------------------------------------------------------- formats --
def quantised(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of ``head_dim`` as e4m3, and for each 32 elements the code c of their scale
    2^(c-127), the smallest under which none of them passes e4m3's largest value, 448."""
    d = x.shape[-1]
    blocks = -(-d // 32)
    xb = torch.nn.functional.pad(x.float(), (0, 32 * blocks - d)).unflatten(-1, (blocks, 32))
    mant, expo = torch.frexp(xb.abs().amax(-1))  # amax = mant * 2^expo, mant in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(mant > 0.875, expo - 8, expo - 9).clamp(min=-126)
    q = torch.ldexp(xb, -e[..., None]).flatten(-2)[..., :d].to(torch.float8_e4m3fn)
    return q, (e + 127).to(torch.uint8)


def values_of(q: torch.Tensor, scales: torch.Tensor | None, to=torch.float32) -> torch.Tensor:
    """What stored rows stand for."""
    x = q.to(to)
    if scales is None:
        return x
    s = torch.ldexp(torch.ones((), dtype=to, device=x.device), scales.to(torch.int32) - 127)
    return x * s.repeat_interleave(32, -1)[..., : x.shape[-1]]


# ------------------------------------------------------------------- prepare --
def prepare(case, seed) -> dict:
    dtype, dev = DTYPES[case["dtype"]], DEVICE
    n, d, page, kvh = case["batch"], case["head_dim"], case["page"], case["kv_heads"]
    lens, news = lengths(case)
    gen = torch.Generator(device=dev).manual_seed(seed * 7919 + 17)
    rnd = lambda *shape: torch.randn(*shape, generator=gen, device=dev)  # noqa: E731
    per = [-(-v // page) for v in lens]
    width, held = max(per), sum(per)
    pool = held + max(4, held // 16)  # a program's pool has pages to spare
    order = torch.randperm(pool, generator=gen, device=dev)[:held].to(torch.int32)
    table = torch.full((n, width), -1, dtype=torch.int32, device=dev)
    table[torch.arange(width, device=dev) < torch.tensor(per, device=dev)[:, None]] = order
    # Keys with a few strong channels, as rotated keys have; values without.
    channel = torch.ones(d, device=dev)
    channel[torch.randperm(d, generator=gen, device=dev)[:4]] = 4.0
    k, v = torch.empty(pool, kvh, page, d, device=dev, dtype=dtype), torch.empty(pool, kvh, page, d, device=dev, dtype=dtype)
    ks = vs = None
    if case["mx"]:
        k, v = k.to(torch.float8_e4m3fn), v.to(torch.float8_e4m3fn)
        ks = torch.empty(pool, kvh, page, -(-d // 32), device=dev, dtype=torch.uint8)
        vs = torch.empty_like(ks)
    step = max(1, (1 << 27) // (kvh * page * d))
    for i in range(0, pool, step):
        m = min(step, pool - i)
        kk, vv = rnd(m, kvh, page, d) * channel, rnd(m, kvh, page, d) + 0.25
        if case["mx"]:
            for t, s, x in ((k, ks, kk), (v, vs, vv)):
                a, b = quantised(x)
                t[i:i + m].view(torch.uint8).copy_(a.view(torch.uint8))
                s[i:i + m] = b
        else:
            k[i:i + m], v[i:i + m] = kk, vv
    state = {"case": case, "k_pages": k, "v_pages": v, "k_scales": ks, "v_scales": vs, "table": table,
             "seq_lens": torch.tensor(lens, dtype=torch.int32, device=dev), "cu": None}
    tokens, seqs = sum(news), torch.arange(n, device=dev)
    if case["ragged"]:
        ends = torch.tensor([0] + news).cumsum(0)
        state["cu"] = ends.to(dtype=torch.int32, device=dev)
    # Which sequence each new token belongs to, and its place among that sequence's new tokens.
    counts = torch.tensor(news, device=dev)
    state["token_seq"] = seqs.repeat_interleave(counts)
    first = counts.cumsum(0) - counts
    state["token_off"] = torch.arange(tokens, device=dev) - first[state["token_seq"]]
    state["position"] = (state["seq_lens"].long() - counts)[state["token_seq"]] + state["token_off"]
    state["longest"], state["most_new"], state["tokens"] = max(lens), max(news), tokens
    shape = (tokens,) if case["ragged"] else (n, case["new"])
    if case["kind"] != "read":
        state["q"] = (rnd(*shape, case["heads"], d) * 1.5 / channel.mean()).to(dtype)
    if case["kind"] == "write":
        state["k"] = (rnd(*shape, kvh, d) * channel).to(dtype)
        state["v"] = (rnd(*shape, kvh, d) + 0.25).to(dtype)
        inv = ROPE_BASE ** (-torch.arange(0, d, 2, dtype=torch.float64, device=dev) / d)
        angle = torch.arange(case["max_len"], dtype=torch.float64, device=dev)[:, None] * inv
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    return state


# ----------------------------------------------------------------------- run --
def run(state):
    if own:
        return _run_own(state)
    return {"write": _plain_write, "read": _plain_read, "attention": _plain_attention}[state["case"]["kind"]](state)


def _run_own(s):
    import ako_amd as ako

    case = s["case"]
    mx = {"k_scales": s["k_scales"], "v_scales": s["v_scales"], "cu_seqlens": s["cu"]}
    where = (s["k_pages"], s["v_pages"], s["table"], s["seq_lens"])
    many = s["tokens"] if case["ragged"] else case["new"]
    if case["kind"] == "read":
        return ako.paged_read(*where, many, DTYPES[case["dtype"]], **mx)
    if case["kind"] == "write":
        q = ako.rope_qk_paged(s["q"], s["k"], s["v"], s["cos"], s["sin"], *where, case["style"], **mx)
        if case["mx"]:
            return (q, *ako.paged_read(*where, many, DTYPES[case["dtype"]], **mx))
        return q, s["k_pages"], s["v_pages"]
    return ako.paged_attention(s["q"], *where, window=case["window"] or None, sinks=case["sinks"], **mx)


def _slots(s):
    """Page and place in it of every new token."""
    page = s["case"]["page"]
    return s["table"][s["token_seq"], s["position"] // page].long(), s["position"] % page


def _rotated(x, cos, sin, style):
    a, b = x.chunk(2, -1) if style == "neox" else (x[..., 0::2], x[..., 1::2])
    r, i = a * cos - b * sin, a * sin + b * cos
    return torch.cat([r, i], -1) if style == "neox" else torch.stack([r, i], -1).flatten(-2)


def _plain_write(s):
    case, dtype = s["case"], DTYPES[s["case"]["dtype"]]
    pages, at = _slots(s)
    cos, sin = s["cos"][s["position"]][:, None], s["sin"][s["position"]][:, None]
    q = _rotated(s["q"].flatten(0, -3).float(), cos, sin, case["style"]).to(dtype).view(s["q"].shape)
    k, v = _rotated(s["k"].flatten(0, -3).float(), cos, sin, case["style"]), s["v"].flatten(0, -3)
    if not case["mx"]:
        s["k_pages"][pages, :, at], s["v_pages"][pages, :, at] = k.to(dtype), v
        return q, s["k_pages"], s["v_pages"]
    (k8, ks), (v8, vs) = quantised(k), quantised(v)
    s["k_pages"].view(torch.uint8)[pages, :, at] = k8.view(torch.uint8)
    s["v_pages"].view(torch.uint8)[pages, :, at] = v8.view(torch.uint8)
    s["k_scales"][pages, :, at], s["v_scales"][pages, :, at] = ks, vs
    return (q, *_plain_read(s))


def _plain_read(s):
    case, dtype = s["case"], DTYPES[s["case"]["dtype"]]
    pages, at = _slots(s)
    shape = (s["tokens"],) if case["ragged"] else (case["batch"], case["new"])

    def rows(t, scales):
        if scales is None:
            x = t[pages, :, at]
        else:
            x = values_of(t.view(torch.uint8)[pages, :, at].view(t.dtype), scales[pages, :, at])
        return x.to(dtype).view(*shape, case["kv_heads"], case["head_dim"])

    return rows(s["k_pages"], s["k_scales"]), rows(s["v_pages"], s["v_scales"])


def _plain_attention(s):
    case, dtype = s["case"], DTYPES[s["case"]["dtype"]]
    n, kvh, d = case["batch"], case["kv_heads"], case["head_dim"]
    group, new, longest = case["heads"] // kvh, s["most_new"], s["longest"]
    ids = s["table"].clamp(min=0).long()

    def dense(t, scales):  # (n, kv_heads, longest, head_dim), 32 bits
        x = t.view(torch.uint8)[ids].view(t.dtype) if scales is not None else t[ids]
        x = values_of(x, None if scales is None else scales[ids])
        return x.transpose(1, 2).flatten(2, 3)[:, :, :longest]

    q = torch.zeros(n, new, case["heads"], d, device=DEVICE)
    q[s["token_seq"], s["token_off"]] = s["q"].flatten(0, -3).float()
    q = q.view(n, new, kvh, group, d).permute(0, 2, 3, 1, 4).reshape(n, kvh, group * new, d)
    score = torch.matmul(q, dense(s["k_pages"], s["k_scales"]).transpose(-1, -2).contiguous()) * d ** -0.5
    counts = s["seq_lens"] if s["cu"] is None else s["cu"].diff()
    counts = torch.full_like(counts, new) if s["cu"] is None else counts
    pos = (s["seq_lens"] - counts)[:, None] + torch.arange(new, device=DEVICE)
    key = torch.arange(longest, device=DEVICE)
    seen = key <= pos[..., None]
    if case["window"]:
        seen &= (key > pos[..., None] - case["window"]) | (key < case["sinks"])
    score = score.view(n, kvh, group, new, longest).masked_fill_(~seen[:, None, None], float("-inf"))
    score -= score.amax(-1, keepdim=True)
    score.exp_()
    total = score.sum(-1, keepdim=True).flatten(2, 3)
    out = torch.matmul(score.flatten(2, 3), dense(s["v_pages"], s["v_scales"]).contiguous()) / total
    out = out.view(n, kvh, group, new, d).permute(0, 3, 1, 2, 4).reshape(n, new, case["heads"], d)
    return out[s["token_seq"], s["token_off"]].to(dtype).view(s["q"].shape)


# ---------------------------------------------------------------------- work --
def work(case) -> dict:
    lens, news = lengths(case)
    eb = DTYPES[case["dtype"]].itemsize
    d, heads, kvh, w, sinks = case["head_dim"], case["heads"], case["kv_heads"], case["window"], case["sinks"]
    row = kvh * (d + -(-d // 32) if case["mx"] else d * eb)  # one position's stored keys (or values)
    tokens = sum(news)
    if case["kind"] == "read":
        return {"bytes": 2 * tokens * (row + kvh * d * eb), "flops": 0}
    if case["kind"] == "write":
        tables = 2 * min(tokens, case["max_len"]) * (d // 2) * 4
        b = tokens * d * eb * 2 * (heads + kvh) + 2 * tokens * row + tables
        if case["mx"]:
            b += 2 * tokens * (row + kvh * d * eb)  # read back
        return {"bytes": b, "flops": 3 * tokens * d * (heads + kvh)}
    pairs, kept = 0, 0
    for length, m in zip(lens, news):
        first = length - m
        if w:
            lo = max(0, first - w + 1)
            kept += (length - lo) + min(sinks, lo)
            for p in range(first, length):
                low = max(0, p - w + 1)
                pairs += p + 1 - low + min(sinks, low)
        else:
            kept += length
            pairs += m * first + m * (m + 1) // 2
    return {"bytes": 2 * kept * row + 2 * tokens * heads * d * eb, "flops": 4 * d * heads * pairs}


# --------------------------------------------------------------------- exact --
def _nearest_e4m3(x):
    """The value of e4m3 nearest to x (64 bits, |x| <= 448), ties to the even one: steps of 2^(e-3)
    for 2^e <= |x| < 2^(e+1), of 2^-9 below 2^-6."""
    _, e = torch.frexp(x.abs().clamp(min=2.0 ** -6))
    step = torch.exp2((e - 4).double())
    return torch.round(x / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    lens, news = lengths(case)
    page, d, f64 = case["page"], case["head_dim"], torch.float64
    table = s["table"].tolist()

    def stored(t, scales, i, upto):
        """Sequence i's first ``upto`` rows, (upto, kv_heads, head_dim)."""
        ids = torch.tensor(table[i][: -(-upto // page)], device=DEVICE)
        x = t.view(torch.uint8)[ids].view(t.dtype).double() if scales is not None else t[ids].double()
        if scales is not None:
            code = scales[ids].double()
            x = x * torch.exp2(code - 127).unsqueeze(-1).expand(*code.shape, 32).flatten(-2)[..., :d]
        return x.permute(0, 2, 1, 3).reshape(-1, case["kv_heads"], d)[:upto]

    if case["kind"] == "read":
        shape = (s["tokens"],) if case["ragged"] else (case["batch"], case["new"])
        return tuple(torch.cat([stored(t, sc, i, n)[n - m:] for i, (n, m) in enumerate(zip(lens, news))])
                     .view(*shape, case["kv_heads"], d)
                     for t, sc in ((s["k_pages"], s["k_scales"]), (s["v_pages"], s["v_scales"])))
    if case["kind"] == "write":
        pos = torch.cat([torch.arange(n - m, n) for n, m in zip(lens, news)]).to(DEVICE)
        # The tables are inputs: their 32-bit values are taken as they are.
        turn = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]

        def rotate(x):
            x = x.flatten(0, -3).double()
            if case["style"] == "neox":
                z = torch.complex(x[..., : d // 2], x[..., d // 2:]) * turn
                return torch.cat([z.real, z.imag], -1)
            return torch.view_as_real(torch.view_as_complex(x.unflatten(-1, (-1, 2)).contiguous()) * turn).flatten(-2)

        q, k, v = rotate(s["q"]).view(s["q"].shape), rotate(s["k"]), s["v"].flatten(0, -3).double()
        if case["mx"]:
            def held(x):
                out = torch.empty_like(x)
                for b in range(0, d, 32):
                    part = x[..., b:b + 32]
                    scale = torch.exp2(torch.ceil(torch.log2(part.abs().amax(-1, keepdim=True) / 448)))
                    out[..., b:b + 32] = _nearest_e4m3(part / scale) * scale
                return out

            return q, held(k).view(s["k"].shape), held(v).view(s["v"].shape)
        kp, vp = s["k_pages"].double(), s["v_pages"].double()
        t = 0
        for i, (n, m) in enumerate(zip(lens, news)):
            at = torch.arange(n - m, n, device=DEVICE)
            ids = torch.tensor(table[i], device=DEVICE)[at // page]
            kp[ids, :, at % page], vp[ids, :, at % page] = k[t:t + m], v[t:t + m]
            t += m
        return q, kp, vp
    rows = []
    q = s["q"].flatten(0, -3)
    group, t = case["heads"] // case["kv_heads"], 0
    for i, (n, m) in enumerate(zip(lens, news)):
        k, v = stored(s["k_pages"], s["k_scales"], i, n), stored(s["v_pages"], s["v_scales"], i, n)
        at = torch.arange(n - m, n, device=DEVICE)[:, None]
        key = torch.arange(n, device=DEVICE)
        hidden = key > at
        if case["window"]:
            hidden = hidden | ((at - key >= case["window"]) & (key >= case["sinks"]))
        out = torch.empty(m, case["heads"], d, dtype=f64, device=DEVICE)
        for h in range(case["heads"]):
            score = (q[t:t + m, h].double() @ k[:, h // group].T.contiguous()) / math.sqrt(d)
            p = torch.softmax(score.masked_fill(hidden, float("-inf")), -1)
            out[:, h] = p @ v[:, h // group].contiguous()
        rows.append(out)
        t += m
    return torch.cat(rows).view(s["q"].shape)

"""A long-context decode step beside the paged cache, as measurable cases.

Four operators of a step of a model that normalises its queries and keys head
by head, attends to the blocks of a long context that a cheap score selects, and
draws its next tokens:

* norm       RMSNorm of every head of q and k with a weight per element, and RoPE, in
             one pass: as dense tensors, or with the keys and the values stored
             in the pages of a cache (the model's type, or e4m3 with scales);
* means      the mean of the keys of every page that a step completed, in 32 bits;
* select     for each token and key head the blocks (pages) to attend to: the first,
             the last, and those whose mean key has the largest product with the sum of
             the queries that share the key head; ties to the lowest block;
* sparse     attention of a step's tokens over the blocks listed for each;
* sample     a token for each row of logits from a given uniform number, after temperature,
             top-k, top-p and min-p.

``listed()`` gives the fixed cases, ``draw`` one more from the ranges they
stand for, ``prepare`` what a program holds before the call, ``run`` one pass
(``own`` false: elementary torch operations; true: the library's operators),
``work`` the bytes and operations a pass cannot do without and ``exact`` its
results in 64 bits.

Ranges (``draw``): 1-64 sequences, one new token or up to 2048 each (all alike,
or packed one after the other), up to 65536 positions, 4-32 query heads in
groups of 1-8, head sizes of 64-256, pages of 16-128 positions and odd ones, 4-128 selected
blocks, float16 / bfloat16 / float32, pages in that type or in e4m3; logits of 1-256
rows of 1000-262144.
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
EPS = 1e-6
#: Blocks that are always selected: the sequence's first, and the token's own.
FIRST, LAST = 1, 1
#: What the largest listed case of a kind has; no drawn case has more.
MAX_LEN = 65536
MAX_CACHE = 16 * 65536 * 8 * 128
MAX_TOKENS = 8192
MAX_SCORES = 2048 * 8 * 512
MAX_PAIRS = 2048 * 32 * 1024
MAX_LOGITS = 256 * 131072


# --------------------------------------------------------------------- cases --
def cache_case(kind, batch, new, max_len, heads, kv_heads, head_dim, page, dtype, *, mx=False, style="neox",
               ragged=False, count=0):
    return {"kind": kind, "batch": batch, "new": new, "max_len": max_len, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "dtype": dtype, "mx": mx, "style": style, "ragged": ragged, "count": count}


def rope_case(batch, new, heads, kv_heads, head_dim, dtype, *, style="neox"):
    return {"kind": "norm_rope", "batch": batch, "new": new, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "dtype": dtype, "style": style}


def sample_case(rows, vocab, dtype, *, per_row, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, masked=False):
    return {"kind": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "per_row": per_row, "temperature": temperature,
            "top_k": top_k, "top_p": top_p, "min_p": min_p, "masked": masked}


def listed() -> list[dict]:
    return [
        # A batch of prompts through one layer: q and k normed and rotated before dense attention.
        {"name": "norm_rope_prompts", **rope_case(4, 2048, 32, 8, 128, "bfloat16")},
        # A serving batch's decode step: norm, rotate and store one token each.
        {"name": "norm_write_step", **cache_case("norm_write", 64, 1, 640, 32, 8, 128, 64, "float16")},
        # Chunks of prompts and single tokens packed in one step, stored in 8 bits and read back.
        {"name": "norm_write_mx8", **cache_case("norm_write", 16, 1024, 4096, 32, 8, 128, 16, "bfloat16", mx=True, ragged=True)},
        # Four whole prompts just stored: the means of all their pages.
        {"name": "means_prompts", **cache_case("means", 4, 8192, 8192, 8, 8, 128, 64, "bfloat16")},
        # A serving batch's decode step, in which a few sequences fill a page of 8-bit keys.
        {"name": "means_step_mx8", **cache_case("means", 64, 1, 8192, 8, 8, 128, 16, "bfloat16", mx=True)},
        # Long contexts, one token each: 64 of 1024 blocks.
        {"name": "select_step", **cache_case("select", 16, 1, 65536, 32, 8, 128, 64, "bfloat16", count=64)},
        # A chunk of 2048 tokens at the end of a context of 32768: 16 of 512 blocks for each.
        {"name": "select_chunk", **cache_case("select", 1, 2048, 32768, 32, 8, 128, 64, "bfloat16", count=16)},
        # One sequence's step on a context of 16384: latency.
        {"name": "sparse_step_one", **cache_case("sparse", 1, 1, 16384, 32, 8, 128, 64, "float16", count=16)},
        # Long contexts in 8 bits, one token each, 64 of 1024 blocks: cache bytes.
        {"name": "sparse_step_long_mx8", **cache_case("sparse", 16, 1, 65536, 32, 8, 128, 64, "bfloat16", mx=True, count=64)},
        # A chunk of 2048 tokens at the end of a context of 32768, 1024 keys each.
        {"name": "sparse_chunk", **cache_case("sparse", 1, 2048, 32768, 32, 8, 128, 64, "bfloat16", count=16)},
        # One sequence's next token, with the decoder's own vocabulary: the smallest call.
        {"name": "sample_one", **sample_case(1, 32000, "float16", per_row=False, temperature=0.8, top_k=50, top_p=0.95)},
        # A serving batch, every row with settings of its own, some tokens ruled out.
        {"name": "sample_batch", **sample_case(256, 131072, "float32", per_row=True, masked=True)},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    while True:
        kind = rng.choice(["norm_rope", "norm_write", "means", "select", "sparse", "sparse", "sample", "sample"])
        dtype = rng.choice(["float16", "bfloat16", "bfloat16", "float32"])
        if kind == "sample":
            rows, vocab = _log_int(rng, 1, 256), _log_int(rng, 1000, 262144)
            if rows * vocab > MAX_LOGITS:
                continue
            return sample_case(rows, vocab, dtype, per_row=rng.random() < 0.5, masked=rng.random() < 0.5,
                               temperature=rng.choice([0.0, 0.7, 1.0, 1.3]), top_k=rng.choice([0, 0, 1, 40, 1000]),
                               top_p=rng.choice([1.0, 0.95, 0.5]), min_p=rng.choice([0.0, 0.0, 0.05]))
        kv_heads, group = rng.choice([4, 4, 8, 8, 32]), rng.choice([1, 4, 8, 8])
        head_dim, page = rng.choice([64, 80, 128, 128, 256]), rng.choice([16, 16, 32, 64, 64, 128, 7, 24])
        heads, style = min(32, kv_heads * group), rng.choice(["neox", "neox", "interleaved"])
        batch, ragged, mx = _log_int(rng, 1, 64), rng.random() < 0.5, rng.random() < 0.5
        new = rng.choice([1, _log_int(rng, 2, 2048)])
        if batch * new > MAX_TOKENS:
            continue
        if kind == "norm_rope":
            return rope_case(batch, new, heads, kv_heads, head_dim, dtype, style=style)
        if kind == "norm_write":
            case = cache_case(kind, batch, new, new + _log_int(rng, 1, 4096), heads, kv_heads, head_dim, page, dtype,
                              mx=mx, style=style, ragged=ragged)
        elif kind == "means":
            case = cache_case(kind, batch, new, new + _log_int(rng, 1, 4096), kv_heads, kv_heads, head_dim, page, dtype,
                              mx=mx, ragged=ragged)
        else:
            case = cache_case(kind, batch, new, new + _log_int(rng, 1, MAX_LEN - new), heads, kv_heads, head_dim, page,
                              dtype, mx=mx and kind == "sparse", ragged=ragged, count=_log_int(rng, 4, 128))
            top = case["max_len"]
            if kind == "select" and batch * new * kv_heads * (top // page + 1) > MAX_SCORES:
                continue
            if kind == "sparse" and batch * new * heads * min(top, case["count"] * page) > MAX_PAIRS:
                continue
        if batch * case["max_len"] * kv_heads * head_dim <= MAX_CACHE:
            return case


def lengths(case) -> tuple[list[int], list[int]]:
    """Positions held by each sequence after the step, and new tokens of each: the same for every seed."""
    n, new, top = case["batch"], case["new"], case["max_len"]
    rng = random.Random(n * 1000003 + new * 1009 + top)
    if not case["ragged"]:  # new tokens alike; contexts within an eighth of the longest
        return [top - (rng.randrange(max(1, (top - new) // 8 + 1)) if i else 0) for i in range(n)], [new] * n
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


def page_rows(pages, scales, ids):
    """Whole pages in 32 bits."""
    x = pages.view(torch.uint8)[ids].view(pages.dtype) if scales is not None else pages[ids]
    return values_of(x, None if scales is None else scales[ids])


# ------------------------------------------------------------------- prepare --
def _rope_tables(rows: int, d: int):
    inv = ROPE_BASE ** (-torch.arange(0, d, 2, dtype=torch.float64, device=DEVICE) / d)
    angle = torch.arange(rows, dtype=torch.float64, device=DEVICE)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed) -> dict:
    gen = torch.Generator(device=DEVICE).manual_seed(seed * 7919 + 17)
    rnd = lambda *shape: torch.randn(*shape, generator=gen, device=DEVICE)  # noqa: E731
    if case["kind"] == "sample":
        return _prepare_sample(case, gen, rnd)
    dtype, dev, d, heads, kvh = DTYPES[case["dtype"]], DEVICE, case["head_dim"], case["heads"], case["kv_heads"]
    weights = lambda: (1.0 + 0.2 * rnd(d)).to(dtype)  # noqa: E731
    if case["kind"] == "norm_rope":
        lead = (case["batch"], case["new"])
        cos, sin = _rope_tables(case["new"], d)
        return {"case": case, "q": (rnd(*lead, heads, d) * 3).to(dtype), "k": (rnd(*lead, kvh, d) * 2).to(dtype),
                "q_weight": weights(), "k_weight": weights(), "cos": cos, "sin": sin}
    n, page = case["batch"], case["page"]
    lens, news = lengths(case)
    per = [-(-v // page) for v in lens]
    width, held = max(per), sum(per)
    pool = held + max(4, held // 16)  # a program's pool has pages to spare
    order = torch.randperm(pool, generator=gen, device=dev)[:held].to(torch.int32)
    table = torch.full((n, width), -1, dtype=torch.int32, device=dev)
    table[torch.arange(width, device=dev) < torch.tensor(per, device=dev)[:, None]] = order
    # The keys of a page have something in common, as a passage's have, and a few strong channels.
    channel = torch.ones(d, device=dev)
    channel[torch.randperm(d, generator=gen, device=dev)[:4]] = 4.0
    k, v = (torch.empty(pool, kvh, page, d, device=dev, dtype=dtype) for _ in range(2))
    ks = vs = None
    if case["mx"]:
        k, v = k.to(torch.float8_e4m3fn), v.to(torch.float8_e4m3fn)
        ks, vs = (torch.empty(pool, kvh, page, -(-d // 32), device=dev, dtype=torch.uint8) for _ in range(2))
    means = torch.empty(pool, kvh, d, device=dev)
    step = max(1, (1 << 27) // (kvh * page * d))
    for i in range(0, pool, step):
        m = min(step, pool - i)
        kk, vv = (rnd(m, kvh, page, d) + 0.6 * rnd(m, kvh, 1, d)) * channel, rnd(m, kvh, page, d) + 0.25
        if case["mx"]:
            for t, s, x in ((k, ks, kk), (v, vs, vv)):
                a, b = quantised(x)
                t[i:i + m].view(torch.uint8).copy_(a.view(torch.uint8))
                s[i:i + m] = b
        else:
            k[i:i + m], v[i:i + m] = kk, vv
        means[i:i + m] = kk.mean(2)
    state = {"case": case, "k_pages": k, "v_pages": v, "k_scales": ks, "v_scales": vs, "k_means": means, "table": table,
             "seq_lens": torch.tensor(lens, dtype=torch.int32, device=dev), "cu": None}
    if case["ragged"]:
        state["cu"] = torch.tensor([0] + news).cumsum(0).to(dtype=torch.int32, device=dev)
    # Which sequence each new token belongs to, and its position there.
    counts = torch.tensor(news, device=dev)
    state["token_seq"] = torch.arange(n, device=dev).repeat_interleave(counts)
    first = counts.cumsum(0) - counts
    off = torch.arange(sum(news), device=dev) - first[state["token_seq"]]
    state["position"] = (state["seq_lens"].long() - counts)[state["token_seq"]] + off
    state["tokens"] = sum(news)
    state["rows"] = sum(news) if case["ragged"] else case["new"]
    shape = (sum(news),) if case["ragged"] else (n, case["new"])
    if case["kind"] == "norm_write":
        state["q"], state["k"] = (rnd(*shape, heads, d) * 3).to(dtype), (rnd(*shape, kvh, d) * channel * 2).to(dtype)
        state["v"] = (rnd(*shape, kvh, d) + 0.25).to(dtype)
        state["q_weight"], state["k_weight"] = weights(), weights()
        state["cos"], state["sin"] = _rope_tables(case["max_len"], d)
    elif case["kind"] in ("select", "sparse"):
        # Neighbouring tokens ask for similar things.
        alike = rnd(n, heads, d)[state["token_seq"]].view(*shape, heads, d)
        state["q"] = ((alike + 0.7 * rnd(*shape, heads, d)) / channel.mean()).to(dtype)
        if case["kind"] == "sparse":
            state["blocks"] = _plain_select(state)
    return state


def _prepare_sample(case, gen, rnd):
    rows, vocab, dev = case["rows"], case["vocab"], DEVICE
    logits = rnd(rows, vocab) * 2.0
    # Most rows have a few likely continuations, some hardly any preference.
    likely = torch.randint(0, vocab, (rows, 24), generator=gen, device=dev)
    logits.scatter_add_(1, likely, rnd(rows, 24).abs() * 4 + torch.rand(rows, 1, generator=gen, device=dev) * 8)
    if case["masked"]:  # as by a grammar: every other row has most of its tokens ruled out
        ruled_out = torch.rand(rows, vocab, generator=gen, device=dev) < 0.9
        ruled_out[::2] = False
        ruled_out.scatter_(1, likely, False)
        logits.masked_fill_(ruled_out, float("-inf"))
    state = {"case": case, "logits": logits.to(DTYPES[case["dtype"]]),
             "uniform": torch.rand(rows, generator=gen, device=dev)}
    if case["per_row"]:
        pick = lambda values, dtype: torch.tensor(values, device=dev, dtype=dtype)[  # noqa: E731
            torch.randint(0, len(values), (rows,), generator=gen, device=dev)]
        state["temperature"] = pick([0.0, 0.6, 0.8, 1.0, 1.0, 1.2], torch.float32)
        state["top_k"] = pick([0, 0, 0, 20, 50, 1000], torch.int32)
        state["top_p"] = pick([1.0, 1.0, 0.95, 0.9, 0.7], torch.float32)
        state["min_p"] = pick([0.0, 0.0, 0.0, 0.02, 0.1], torch.float32)
    else:
        state.update({name: case[name] for name in ("temperature", "top_k", "top_p", "min_p")})
    return state


# ----------------------------------------------------------------------- run --
def run(state):
    if own:
        return _run_own(state)
    return {"norm_rope": _plain_norm_rope, "norm_write": _plain_norm_write, "means": _plain_means, "select": _plain_select,
            "sparse": _plain_sparse, "sample": _plain_sample}[state["case"]["kind"]](state)


def _run_own(s):
    import ako_amd as ako

    case = s["case"]
    if case["kind"] == "sample":
        return ako.sample(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                          min_p=s["min_p"])
    if case["kind"] == "norm_rope":
        return ako.rmsnorm_rope_qk(s["q"], s["k"], s["q_weight"], s["k_weight"], s["cos"], s["sin"], EPS, case["style"])
    if case["kind"] == "means":
        return ako.paged_means(s["k_pages"], s["k_means"], s["table"], s["seq_lens"], s["rows"], k_scales=s["k_scales"],
                               cu_seqlens=s["cu"])
    if case["kind"] == "select":
        return ako.paged_select(s["q"], s["k_means"], s["table"], s["seq_lens"], case["page"], case["count"], first=FIRST,
                                last=LAST, cu_seqlens=s["cu"])
    where = (s["k_pages"], s["v_pages"], s["table"], s["seq_lens"])
    mx = {"k_scales": s["k_scales"], "v_scales": s["v_scales"], "cu_seqlens": s["cu"]}
    if case["kind"] == "sparse":
        return ako.paged_attention(s["q"], *where, blocks=s["blocks"], **mx)
    q = ako.rope_qk_paged(s["q"], s["k"], s["v"], s["cos"], s["sin"], *where, case["style"], q_weight=s["q_weight"],
                          k_weight=s["k_weight"], eps=EPS, **mx)
    if case["mx"]:
        return (q, *ako.paged_read(*where, s["rows"], DTYPES[case["dtype"]], **mx))
    return q, s["k_pages"], s["v_pages"]


def _normed(x, weight):
    x = x.float()
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()


def _rotated(x, cos, sin, style):
    a, b = x.chunk(2, -1) if style == "neox" else (x[..., 0::2], x[..., 1::2])
    r, i = a * cos - b * sin, a * sin + b * cos
    return torch.cat([r, i], -1) if style == "neox" else torch.stack([r, i], -1).flatten(-2)


def _plain_norm_rope(s):
    cos, sin, style = s["cos"][:, None], s["sin"][:, None], s["case"]["style"]
    return tuple(_rotated(_normed(x, w), cos, sin, style).to(x.dtype)
                 for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])))


def _plain_norm_write(s):
    case, dtype, at = s["case"], DTYPES[s["case"]["dtype"]], s["position"] % s["case"]["page"]
    pages = s["table"][s["token_seq"], s["position"] // case["page"]].long()
    cos, sin = s["cos"][s["position"]][:, None], s["sin"][s["position"]][:, None]
    q, k = (_rotated(_normed(x.flatten(0, -3), w), cos, sin, case["style"])
            for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])))
    q, v = q.to(dtype).view(s["q"].shape), s["v"].flatten(0, -3)
    if not case["mx"]:
        s["k_pages"][pages, :, at], s["v_pages"][pages, :, at] = k.to(dtype), v
        return q, s["k_pages"], s["v_pages"]
    out = [q]
    for t, codes, x in ((s["k_pages"], s["k_scales"], k), (s["v_pages"], s["v_scales"], v)):
        x8, c = quantised(x)
        t.view(torch.uint8)[pages, :, at], codes[pages, :, at] = x8.view(torch.uint8), c
        x8, c = t.view(torch.uint8)[pages, :, at].view(t.dtype), codes[pages, :, at]
        out.append(values_of(x8, c).to(dtype).view(s["k"].shape))
    return tuple(out)


def _plain_means(s):
    full = (s["position"] + 1) % s["case"]["page"] == 0  # the tokens that fill their page
    pages = s["table"][s["token_seq"][full], s["position"][full] // s["case"]["page"]].long()
    s["k_means"][pages] = page_rows(s["k_pages"], s["k_scales"], pages).mean(2)
    return s["k_means"]


def _plain_select(s):
    """In 64 bits: which of two blocks comes first hangs on the last bits of their scores."""
    case, page, kvh, count = s["case"], s["case"]["page"], s["case"]["kv_heads"], s["case"]["count"]
    q = s["q"].flatten(0, -3).double().unflatten(1, (kvh, -1)).sum(2)  # (tokens, kv_heads, head_dim)
    own_block, width = s["position"] // page, s["table"].shape[1]
    block = torch.arange(width, device=DEVICE)
    score = torch.empty(s["tokens"], kvh, width, dtype=torch.float64, device=DEVICE)
    ids, at = s["table"].clamp(min=0).long(), 0
    for i, m in enumerate(lengths(case)[1]):
        mean = s["k_means"][ids[i]].double().permute(1, 2, 0).contiguous()  # (kv_heads, head_dim, width)
        score[at:at + m] = torch.matmul(q[at:at + m].transpose(0, 1).contiguous(), mean).transpose(0, 1)
        at += m
    own_block = own_block[:, None, None]
    score.masked_fill_((block < FIRST) | (block > own_block - LAST), float("inf")).masked_fill_(block > own_block, float("-inf"))
    best, where = torch.sort(score, dim=-1, descending=True, stable=True)  # of equal ones the lowest block first
    best, where = best[..., :count], where[..., :count]
    where = torch.where(best == float("-inf"), width, where).sort(-1).values
    if where.shape[-1] < count:
        where = torch.nn.functional.pad(where, (0, count - where.shape[-1]), value=width)
    return torch.where(where == width, -1, where).to(torch.int32).view(*s["q"].shape[:-2], kvh, count)


def _plain_sparse(s):
    case, kvh, d, page, count = s["case"], s["case"]["kv_heads"], s["case"]["head_dim"], s["case"]["page"], s["case"]["count"]
    q = s["q"].flatten(0, -3)
    group, out = case["heads"] // kvh, torch.empty_like(q)
    blocks = s["blocks"].flatten(0, -3).long()  # (tokens, kv_heads, count)
    head = torch.arange(kvh, device=DEVICE)[:, None]
    step = max(1, (1 << 28) // (kvh * count * page * d))
    for t in range(0, s["tokens"], step):
        b, pos = blocks[t:t + step], s["position"][t:t + step, None, None, None]
        ids = s["table"][s["token_seq"][t:t + step, None, None], b.clamp(min=0)].long()

        def rows(pages, scales):  # (tokens, kv_heads, count * page, head_dim), 32 bits
            x = pages.view(torch.uint8)[ids, head].view(pages.dtype) if scales is not None else pages[ids, head]
            return values_of(x, None if scales is None else scales[ids, head]).flatten(2, 3)

        key = b[..., None] * page + torch.arange(page, device=DEVICE)
        seen = ((key <= pos) & (b >= 0)[..., None]).flatten(2)
        x = q[t:t + step].float().unflatten(1, (kvh, group))
        score = torch.matmul(x, rows(s["k_pages"], s["k_scales"]).transpose(-1, -2).contiguous()) * d ** -0.5
        score.masked_fill_(~seen[:, :, None], float("-inf"))
        p = torch.exp(score - score.amax(-1, keepdim=True))
        o = torch.matmul(p, rows(s["v_pages"], s["v_scales"])) / p.sum(-1, keepdim=True)
        out[t:t + step] = o.flatten(1, 2).to(q.dtype)
    return out.view(s["q"].shape)


def _column(value, rows, dtype):
    if torch.is_tensor(value):
        return value[:, None].to(dtype)
    return torch.full((rows, 1), value, device=DEVICE, dtype=torch.float32).to(dtype)


def _plain_sample(s):
    """In 64 bits: sums over a whole vocabulary are compared with a number that falls between two of its tokens."""
    x = s["logits"].double()
    rows, vocab = x.shape
    f64 = torch.float64
    t, p, low = (_column(s[name], rows, f64) for name in ("temperature", "top_p", "min_p"))
    k = _column(s["top_k"], rows, torch.int64)
    top = x.amax(-1, keepdim=True)
    w = torch.exp((x - top) / torch.where(t > 0, t, 1.0))
    ordered, index = torch.sort(x, dim=-1, descending=True, stable=True)  # of equal ones the lowest index first
    wo = torch.gather(w, 1, index)
    rank = torch.arange(vocab, device=DEVICE)
    wo = wo.masked_fill((k > 0) & (rank >= k), 0.0)
    before = wo.cumsum(-1) - wo
    keep = (wo > 0) & ((before < p * wo.sum(-1, keepdim=True)) | (p >= 1)) & (wo >= low) | (rank == 0)
    keep &= (t > 0) | (rank == 0)
    kept = torch.zeros_like(w).scatter_(1, index, torch.where(keep, wo, 0.0)).cumsum(-1)
    target = s["uniform"].double()[:, None] * kept[:, -1:]
    return torch.searchsorted(kept, target, right=True)[:, 0]


# ---------------------------------------------------------------------- work --
def work(case) -> dict:
    eb = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * eb + case["rows"] * (28 if case["per_row"] else 12), "flops": 4 * n}
    d, heads, kvh = case["head_dim"], case["heads"], case["kv_heads"]
    if case["kind"] == "norm_rope":
        n = case["batch"] * case["new"] * (heads + kvh) * d
        return {"bytes": 2 * n * eb + case["new"] * d * 4 + 2 * d * eb, "flops": 7 * n}
    lens, news = lengths(case)
    page, count, tokens = case["page"], case["count"], sum(news)
    row = kvh * (d + -(-d // 32) if case["mx"] else d * eb)  # one position's stored keys (or values)
    if case["kind"] == "norm_write":
        b = tokens * d * eb * 2 * (heads + kvh) + 2 * tokens * row + min(tokens, case["max_len"]) * d * 4
        if case["mx"]:
            b += 2 * tokens * (row + kvh * d * eb)  # read back
        return {"bytes": b, "flops": 7 * tokens * d * (heads + kvh)}
    if case["kind"] == "means":
        full = sum(n // page - (n - m) // page for n, m in zip(lens, news))
        return {"bytes": full * (page * row + kvh * d * 4), "flops": full * page * kvh * d}
    if case["kind"] == "select":
        scores = sum(p // page for n, m in zip(lens, news) for p in range(n - m, n))
        held = sum(n // page for n in lens)
        return {"bytes": tokens * (heads * d * eb + kvh * count * 4) + held * kvh * d * 4,
                "flops": 2 * scores * kvh * d + tokens * heads * d}
    pairs = moved = 0
    for n, m in zip(lens, news):
        seen = [min(p // page + 1, count) * page - (page - 1 - p % page) for p in range(n - m, n)]
        pairs += sum(seen)
        moved += min(n, sum(seen))
    return {"bytes": 2 * moved * row + 2 * tokens * heads * d * eb + tokens * kvh * count * 4, "flops": 4 * d * heads * pairs}


# --------------------------------------------------------------------- exact --
def _nearest_e4m3(x):
    """The value of e4m3 nearest to x (64 bits, |x| <= 448), ties to the even one: steps of 2^(e-3)
    for 2^e <= |x| < 2^(e+1), of 2^-9 below 2^-6."""
    _, e = torch.frexp(x.abs().clamp(min=2.0 ** -6))
    step = torch.exp2((e - 4).double())
    return torch.round(x / step) * step


def _held(x):
    """What 8-bit rows with block scales hold of x."""
    out = torch.empty_like(x)
    for b in range(0, x.shape[-1], 32):
        part = x[..., b:b + 32]
        scale = torch.exp2(torch.ceil(torch.log2(part.abs().amax(-1, keepdim=True) / 448)))
        out[..., b:b + 32] = _nearest_e4m3(part / scale) * scale
    return out


def _exact_turn(x, weight, turn, style):
    """RMSNorm over the last dimension, then every pair as a complex number times ``turn``."""
    d = x.shape[-1]
    x = x.double()
    x = x / torch.sqrt(torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / d + EPS) * weight.double()
    if style == "neox":
        z = torch.complex(x[..., : d // 2], x[..., d // 2:]) * turn
        return torch.cat([z.real, z.imag], -1)
    return torch.view_as_real(torch.view_as_complex(x.unflatten(-1, (-1, 2)).contiguous()) * turn).flatten(-2)


def _exact_rows(s, pages, scales, i, upto):
    """Sequence i's first ``upto`` stored rows, (kv_heads, upto, head_dim)."""
    ids = s["table"][i, : -(-upto // s["case"]["page"])].long()
    if scales is None:
        x = pages[ids].double()
    else:
        x = pages.view(torch.uint8)[ids].view(pages.dtype).double()
        x = x * torch.exp2(scales[ids].double() - 127).unsqueeze(-1).expand(*scales[ids].shape, 32).flatten(-2)[..., : x.shape[-1]]
    return x.transpose(0, 1).flatten(1, 2)[:, :upto]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "sample":
        return _exact_sample(s)
    if case["kind"] == "norm_rope":
        turn = torch.complex(s["cos"].double(), s["sin"].double())[:, None]
        return tuple(_exact_turn(s[x], s[x + "_weight"], turn, case["style"]) for x in "qk")
    lens, news = lengths(case)
    page, kvh, d = case["page"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "norm_write":
        pos = torch.cat([torch.arange(n - m, n) for n, m in zip(lens, news)]).to(DEVICE)
        turn = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]
        q, k = (_exact_turn(s[x].flatten(0, -3), s[x + "_weight"], turn, case["style"]) for x in "qk")
        v, q = s["v"].flatten(0, -3).double(), q.view(s["q"].shape)
        if case["mx"]:
            return q, _held(k).view(s["k"].shape), _held(v).view(s["v"].shape)
        kp, vp, t = s["k_pages"].double(), s["v_pages"].double(), 0
        for i, (n, m) in enumerate(zip(lens, news)):
            at = torch.arange(n - m, n, device=DEVICE)
            ids = s["table"][i].long()[at // page]
            kp[ids, :, at % page], vp[ids, :, at % page] = k[t:t + m], v[t:t + m]
            t += m
        return q, kp, vp
    if case["kind"] == "means":
        out = s["k_means"].double()
        for i, (n, m) in enumerate(zip(lens, news)):
            lo, hi = (n - m) // page, n // page  # the pages that positions n - m .. n - 1 fill
            if hi > lo:
                keys = _exact_rows(s, s["k_pages"], s["k_scales"], i, hi * page)[:, lo * page:]
                out[s["table"][i, lo:hi].long()] = keys.unflatten(1, (-1, page)).sum(2).transpose(0, 1) / page
        return out
    group = case["heads"] // kvh
    q, t, parts = s["q"].flatten(0, -3).double(), 0, []
    if case["kind"] == "select":
        for i, (n, m) in enumerate(zip(lens, news)):
            mean = s["k_means"].double()[s["table"][i, : -(-n // page)].long()]
            for h in range(kvh):
                # One head at a time, and the heads' scores added up.
                score = sum(q[t:t + m, h * group + g] @ mean[:, h].T.contiguous() for g in range(group))
                mine = (torch.arange(n - m, n, device=DEVICE) // page)[:, None]
                b = torch.arange(score.shape[1], device=DEVICE)
                always = (b < FIRST) | (b > mine - LAST)
                # 0: always taken, 1: by score, 2: not there yet; then by score, then by number.
                order = torch.argsort(-score, dim=-1, stable=True)
                rank = torch.where(b > mine, 2, torch.where(always, 0, 1)).gather(1, order)
                order = order.gather(1, torch.argsort(rank, dim=-1, stable=True))
                chosen = torch.zeros_like(score, dtype=torch.bool).scatter_(1, order[:, : case["count"]], True) & (b <= mine)
                row = torch.full((m, case["count"]), -1, dtype=torch.int32, device=DEVICE)
                r, c = chosen.nonzero(as_tuple=True)
                row[r, chosen.cumsum(1)[r, c] - 1] = c.int()
                parts.append((t, m, h, row))
            t += m
        out = torch.empty(s["tokens"], kvh, case["count"], dtype=torch.int32, device=DEVICE)
        for t, m, h, row in parts:
            out[t:t + m, h] = row
        return out.view(*s["q"].shape[:-2], kvh, case["count"])
    blocks = s["blocks"].flatten(0, -3).long()
    out = torch.empty_like(q)
    for i, (n, m) in enumerate(zip(lens, news)):
        k, v = _exact_rows(s, s["k_pages"], s["k_scales"], i, n), _exact_rows(s, s["v_pages"], s["v_scales"], i, n)
        for a in range(0, m, 256):  # over all keys, those of other blocks hidden
            c = min(256, m - a)
            at = torch.arange(n - m + a, n - m + a + c, device=DEVICE)[:, None]
            key = torch.arange(n, device=DEVICE)
            for h in range(kvh):
                taken = torch.zeros(c, -(-n // page) + 1, dtype=torch.bool, device=DEVICE)
                taken.scatter_(1, blocks[t + a:t + a + c, h] % taken.shape[1], True)  # -1: the last column
                hidden = ~taken[:, :-1].repeat_interleave(page, 1)[:, :n] | (key > at)
                for g in range(h * group, (h + 1) * group):
                    score = (q[t + a:t + a + c, g] @ k[h].T.contiguous()) / math.sqrt(d)
                    out[t + a:t + a + c, g] = torch.softmax(score.masked_fill(hidden, float("-inf")), -1) @ v[h]
        t += m
    return out.view(s["q"].shape)


def _exact_sample(s):
    """Row by row, from the logits alone."""
    value = lambda name, r: float(s[name][r]) if torch.is_tensor(s[name]) else float(torch.tensor(s[name], dtype=torch.float32))  # noqa: E731
    out = []
    for r in range(s["logits"].shape[0]):
        x = s["logits"][r].double()
        t, k, p, low = (value(name, r) for name in ("temperature", "top_k", "top_p", "min_p"))
        order = torch.argsort(-x, stable=True)
        order = order[x[order] > float("-inf")]
        if k > 0:
            order = order[: int(k)]
        if t <= 0:
            order = order[:1]
        z = (x[order] - x[order[0]]) / (t if t > 0 else 1.0)
        share = torch.softmax(z, 0)
        n = order.numel()
        if p < 1:  # the fewest that reach p
            n = max(1, min(n, int((share.cumsum(0) < p).sum()) + 1))
        if low > 0:
            n = max(1, min(n, int((z >= math.log(low)).sum())))
        index, by = order[:n].sort()
        total = torch.exp(z[:n][by]).cumsum(0)
        out.append(index[int((total <= float(s["uniform"][r]) * total[-1]).sum().clamp(max=n - 1))])
    return torch.stack(out)

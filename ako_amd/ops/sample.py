"""Drawing a token for each row of logits from a given uniform number.

With ``w = exp((logits - max) / temperature)``, and the tokens in descending
order of their logits, of equal ones the lowest index first:

* ``top_k`` keeps the first ``top_k`` of them (0: all);
* ``top_p`` keeps, of those, the shortest run from the front that weighs at least
  ``top_p`` of them all, one token at least (1: all);
* ``min_p`` keeps, of those, the tokens with ``w >= min_p`` (0: all).

The token drawn is the first, by index, at which the sum of the kept weights so far
passes ``uniform`` times their whole sum. ``temperature`` 0 takes the first token
of the largest logit. Tokens of -infinity or NaN are never drawn; a row of nothing else
gives -1. Where logits are +infinity only those tokens are drawn, all alike.

Every setting is one number, or a tensor of one for each row, which a captured call
follows. In tensors, whose values the host does not see, temperatures below 0 or NaN count as 0,
``top_k`` below 0 as 0, ``top_p`` above 1 or NaN as 1 and below 0 as 0, ``min_p`` below 0 or
NaN as 0 and above 1 as 1; uniform numbers below 0 or NaN count as 0, and from 1 on they give the last
token kept.

On a GPU this runs the HIP kernel (and raises if the library cannot be loaded,
unless ``AKO_HIP_DISABLE=1``), on a CPU the sorts below. The kernel's weights are whole
multiples of 2^-51 of the largest (2^-45 at 131072 tokens), and what is below half of that is ruled
out; its token does not depend on the batch around a row.
"""

from __future__ import annotations

import math

import torch

from ako_amd import _native
from ako_amd.ops._hip_common import DT, call, gpu_index, lib, raw_stream
from ako_amd.ops._registry import hip_disabled

MAX_VOCAB = 1 << 22


def sample(
    logits: torch.Tensor,
    uniform: torch.Tensor,
    *,
    temperature: float | torch.Tensor = 1.0,
    top_k: int | torch.Tensor = 0,
    top_p: float | torch.Tensor = 1.0,
    min_p: float | torch.Tensor = 0.0,
) -> torch.Tensor:
    """A token for each row of ``logits (rows, vocab)`` from ``uniform (rows,)``, float32 in [0, 1); int64.

    Settings per row are float32 tensors, ``top_k`` an int32 one.
    """
    if logits.is_cuda and not hip_disabled():
        return sample_hip(logits, uniform, temperature, top_k, top_p, min_p)
    return sample_ref(logits, uniform, temperature, top_k, top_p, min_p)


def sample_error(logits, uniform, temperature, top_k, top_p, min_p) -> str | None:
    """The first thing wrong with a call's arguments, or ``None``."""
    if logits.dim() != 2:
        return f"logits must be (rows, vocab), got {tuple(logits.shape)}"
    if logits.dtype not in DT:
        return f"logits must be float32/float16/bfloat16, got {logits.dtype}"
    rows, vocab = logits.shape
    if not 1 <= vocab <= MAX_VOCAB:
        return f"vocab must be 1 to {MAX_VOCAB}, got {vocab}"

    def row_error(name, t, dtype, kind):
        if tuple(t.shape) != (rows,) or t.dtype != dtype or not t.is_contiguous() or t.device != logits.device:
            return f"{name} must be {kind}a contiguous {dtype} tensor of shape ({rows},) on the device of the logits"
        return None

    wrong = row_error("uniform", uniform, torch.float32, "")
    settings = {"temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p}
    for name, v in settings.items():
        if wrong is None and torch.is_tensor(v):
            wrong = row_error(name, v, torch.int32 if name == "top_k" else torch.float32, "a number or ")
    if wrong:
        return wrong
    if not torch.is_tensor(temperature) and not temperature >= 0:
        return f"temperature must be at least 0, got {float(temperature)}"
    if not torch.is_tensor(top_k) and not (top_k >= 0 and math.isfinite(top_k) and top_k == math.floor(top_k)):
        return f"top_k must be a whole number, at least 0, got {top_k}"
    for name in ("top_p", "min_p"):
        v = settings[name]
        if not torch.is_tensor(v) and not 0 <= v <= 1:
            return f"{name} must be 0 to 1, got {float(v)}"
    return None


def _refuse(fn_name: str, *args) -> None:
    wrong = sample_error(*args)
    if wrong:
        raise ValueError(f"{fn_name}: {wrong}")


def sample_ref(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> torch.Tensor:
    """In 64 bits, by sorting."""
    _refuse("sample", logits, uniform, temperature, top_k, top_p, min_p)
    rows, vocab = logits.shape

    def column(v, dtype=torch.float32):
        if not torch.is_tensor(v):  # numbers past float32's largest are infinite, as for the kernel
            v = torch.full((rows,), min(v, 2**31 - 1) if dtype != torch.float32 else v, dtype=torch.float64, device=logits.device).to(dtype)
        return v[:, None].double() if dtype == torch.float32 else v[:, None].long()

    t, k, p, low = column(temperature), column(top_k, torch.int32), column(top_p), column(min_p)
    x = logits.double()
    x = torch.where(x.isnan(), -math.inf, x)
    live = x > -math.inf
    top = x.amax(-1, keepdim=True)
    draw = (t > 0) & live.any(-1, keepdim=True)
    w = torch.exp((x - top) / torch.where(draw, t, 1.0))
    w = torch.where(x == top, 1.0, torch.where(live, w, 0.0)).nan_to_num(0.0)
    ordered, index = torch.sort(torch.where(live, x, -math.inf), dim=-1, descending=True, stable=True)
    wo = torch.gather(w, 1, index)
    rank = torch.arange(vocab, device=x.device)
    wo = wo.masked_fill((k > 0) & (rank >= k), 0.0)
    before = wo.cumsum(-1) - wo
    keep = (before < p * wo.sum(-1, keepdim=True)) | ~(p < 1)
    keep &= (wo >= low.clamp(max=1.0)) | ~(low > 0)
    keep &= ~(low >= 1) | (torch.gather(x, 1, index) == top)  # next to the largest weights round to 1
    keep = torch.where(draw, (keep & (wo > 0)) | (rank == 0), rank == 0)
    kept = torch.zeros_like(w).scatter_(1, index, torch.where(keep, wo, 0.0))
    upto = kept.cumsum(-1)
    u = uniform.double()[:, None]
    token = torch.searchsorted(upto, torch.where(u > 0, u, 0.0) * upto[:, -1:], right=True)[:, 0]
    last = vocab - 1 - (kept > 0).flip(-1).int().argmax(-1)
    return torch.where(live.any(-1), torch.minimum(token, last), -1)


def sample_hip(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> torch.Tensor:
    fast = _native.torch_binding()
    if fast is not None:
        return fast.sample(logits, uniform, temperature, top_k, top_p, min_p)
    return sample_hip_ctypes(logits, uniform, temperature, top_k, top_p, min_p)


def sample_hip_ctypes(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> torch.Tensor:
    fn = "sample_hip"
    index = gpu_index(logits, fn)
    _refuse(fn, logits, uniform, temperature, top_k, top_p, min_p)
    rows, vocab = logits.shape
    x = logits if logits.stride(1) == 1 or vocab == 1 else logits.contiguous()
    out = torch.empty(rows, dtype=torch.int64, device=logits.device)
    both = lambda v, none: (v.data_ptr(), none) if torch.is_tensor(v) else (None, v)  # noqa: E731
    need = max(0, lib().ako_sample_workspace(rows, vocab, DT[logits.dtype]))
    space = torch.empty(need, dtype=torch.uint8, device=logits.device) if need else None
    top_k = top_k if torch.is_tensor(top_k) else min(int(top_k), 2**31 - 1)
    status = call(index, lib().ako_sample_fwd, x.data_ptr(), uniform.data_ptr(), *both(temperature, 0.0), *both(top_k, 0),
                  *both(top_p, 0.0), *both(min_p, 0.0), out.data_ptr(), rows, vocab, x.stride(0) if rows > 1 else vocab,
                  space.data_ptr() if need else None, need, DT[logits.dtype], raw_stream(index))
    if status:
        _native.check(status, fn)
    return out


__all__ = ["sample"]

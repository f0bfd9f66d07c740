"""RMSNorm of every head of q and k with RoPE in the same pass.

Models that normalise their queries and keys head by head do so right before the
rotation. ``rmsnorm_rope_qk`` is both, as dense tensors; with a paged cache
``rope_qk_paged`` takes the same weights and stores the keys as it goes. Nothing is
rounded between the norm and the rotation. Like the cache operations it is called directly:
on a GPU it runs the HIP kernel (and raises if the library cannot be loaded, unless
``AKO_HIP_DISABLE=1``), on a CPU the composition below.
"""

from __future__ import annotations

import ctypes
import warnings

import torch

from ako_amd import _native
from ako_amd.ops._hip_common import DT, call, gpu_index, lib, raw_stream
from ako_amd.ops._registry import hip_disabled
from ako_amd.ops.rmsnorm_ref import rmsnorm_ref
from ako_amd.ops.rope_hip import _head_view, _table, _table_stride
from ako_amd.ops.rope_ref import rope_ref, validate_rope_args

#: The largest head that one wavefront normalises.
MAX_HEAD_DIM = 512

_I64x3 = ctypes.c_int64 * 3


def rmsnorm_rope_qk(
    q: torch.Tensor,
    k: torch.Tensor,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    eps: float = 1e-6,
    style: str = "neox",
) -> tuple[torch.Tensor, torch.Tensor]:
    """``rope(rmsnorm(q, q_weight))`` and ``rope(rmsnorm(k, k_weight))`` over heads.

    q and k are ``(batch, seq, heads, head_dim)`` with head counts of their own, the
    weights ``(head_dim,)``, ``cos``/``sin`` the ``(seq, head_dim / 2)`` rows of the
    positions. ``head_dim`` is even, at most 512. There is no backward pass: on a GPU
    the results carry no gradient, with a warning where one could be expected of them.
    """
    args = (q, k, q_weight, k_weight, cos, sin, eps, style)
    if q.is_cuda and not hip_disabled():
        if torch.is_grad_enabled() and any(t.requires_grad for t in args[:4]):
            warnings.warn("rmsnorm_rope_qk has no backward pass on a GPU: no gradient goes from its results to q, k "
                          "or the weights; call it under torch.no_grad() where none is wanted", stacklevel=2)
        return rmsnorm_rope_qk_hip(*args)
    return rmsnorm_rope_qk_ref(*args)


def weights_error(q_weight, k_weight, eps, head_dim: int, like: torch.Tensor) -> str | None:
    """The first thing wrong with the weights of the heads' norms, or ``None``."""
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if tuple(w.shape) != (head_dim,):
            return f"Expected {name} of shape ({head_dim},), got {tuple(w.shape)}"
        if w.device != like.device:
            return f"{name} must be on the device of q"
    if not eps >= 0:
        return f"eps must be at least 0, got {eps}"
    return None


def kernel_weights(q_weight: torch.Tensor, k_weight: torch.Tensor, dtype: torch.dtype):
    """Both weights as the kernels take them: of the rows' type, or else of float32."""
    if q_weight.dtype != dtype or k_weight.dtype != dtype:
        q_weight, k_weight = q_weight.float(), k_weight.float()
    return q_weight.contiguous(), k_weight.contiguous()


def _check(fn_name, q, k, q_weight, k_weight, cos, sin, eps, style) -> None:
    validate_rope_args(q, cos, sin, style)
    validate_rope_args(k, cos, sin, style)
    wrong = None
    if q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3] or q.dtype != k.dtype or q.device != k.device:
        wrong = f"q {tuple(q.shape)} {q.dtype} and k {tuple(k.shape)} {k.dtype} must match but for their heads"
    elif q.dtype not in DT:
        wrong = f"q must be float32/float16/bfloat16, got {q.dtype}"
    elif not 2 <= q.shape[3] <= MAX_HEAD_DIM:
        wrong = f"head_dim must be 2 to {MAX_HEAD_DIM}, got {q.shape[3]}"
    wrong = wrong or weights_error(q_weight, k_weight, eps, q.shape[3], q)
    if wrong is None and (cos.device != q.device or sin.device != q.device):
        wrong = "tables must be on the device of q"
    if wrong:
        raise ValueError(f"{fn_name}: {wrong}")


def norm_rope_rows(x: torch.Tensor, weight: torch.Tensor, cos, sin, eps: float, style: str) -> torch.Tensor:
    """Normed and rotated heads in 32 bits, not rounded to a shorter type."""
    return rope_ref(rmsnorm_ref(x.float(), weight, eps), cos, sin, style)


def rmsnorm_rope_qk_ref(q, k, q_weight, k_weight, cos, sin, eps=1e-6, style="neox"):
    _check("rmsnorm_rope_qk", q, k, q_weight, k_weight, cos, sin, eps, style)
    return tuple(norm_rope_rows(x, w, cos, sin, eps, style).to(x.dtype) for x, w in ((q, q_weight), (k, k_weight)))


def rmsnorm_rope_qk_hip(q, k, q_weight, k_weight, cos, sin, eps=1e-6, style="neox"):
    """Both tensors in one launch."""
    fast = _native.torch_binding()
    if fast is not None:
        return fast.rmsnorm_rope_qk(q, k, q_weight, k_weight, cos, sin, eps, style)
    return rmsnorm_rope_qk_hip_ctypes(q, k, q_weight, k_weight, cos, sin, eps, style)


def rmsnorm_rope_qk_hip_ctypes(q, k, q_weight, k_weight, cos, sin, eps=1e-6, style="neox"):
    fn = "rmsnorm_rope_qk_hip"
    index = gpu_index(q, fn)
    _check(fn, q, k, q_weight, k_weight, cos, sin, eps, style)
    qv, kv = _head_view(q), _head_view(k)
    qw, kw = kernel_weights(q_weight, k_weight, q.dtype)
    c, s, st = _table_stride(_table(cos, index), _table(sin, index))
    q_out, k_out = (torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, k))
    batch, seq, heads, head_dim = q.shape
    status = call(index, lib().ako_rmsnorm_rope_qk_fwd, qv.data_ptr(), kv.data_ptr(), qw.data_ptr(), kw.data_ptr(),
                  c.data_ptr(), s.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), batch, seq, heads, k.shape[2], head_dim,
                  _I64x3(*qv.stride()[:3]), _I64x3(*kv.stride()[:3]), st, eps, DT[q.dtype], DT[qw.dtype], DT[c.dtype],
                  _native.ROPE_STYLE_CODES[style], raw_stream(index))
    if status:
        _native.check(status, fn)
    return q_out, k_out


__all__ = ["rmsnorm_rope_qk"]

"""Calls of the paged-cache operations at the ends of what their documentation allows: no query heads, no
pages, no table, rows and tables as views."""

from __future__ import annotations

import pytest
import torch

import ako_amd as ako
from tests._paged import E4M3, attention64, step, tables
from tests.test_paged_nonfinite import DEVICES, assert_same, results


def check(s, **opts) -> None:
    want, bound = attention64(s, **opts)
    for name, out in results(s, **opts):
        assert_same(out, want, bound, name)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("mx", [False, True])
def test_no_query_heads(mx: bool, packed: bool, device: str) -> None:
    """Keys and values are stored all the same."""
    s = step([20, 9], [3, 3], dtype=torch.float16, mx=mx, packed=packed, device=device)
    cos, sin = tables(30, 64, device)
    want = step([20, 9], [3, 3], dtype=torch.float16, mx=mx, packed=packed, device=device)
    ako.rope_qk_paged(want.q, want.k, want.v, cos, sin, *want.where, **want.kw)
    q = s.q[..., :0, :]
    assert ako.rope_qk_paged(q, s.k, s.v, cos, sin, *s.where, **s.kw).shape == q.shape
    assert ako.paged_attention(q, *s.where, **s.kw).shape == q.shape
    for a, b in zip(ako.paged_read(*s.where, s.rows, torch.float16, **s.kw), ako.paged_read(*want.where, s.rows, torch.float16, **want.kw)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float16, E4M3])
def test_a_pool_without_pages_and_a_table_without_columns(dtype, device: str) -> None:
    kp, vp, ks, vs = ako.new_pages(0, 2, 16, 64, dtype, device=device)
    s = step([20, 9], [3, 3], dtype=torch.float16, mx=dtype == E4M3, device=device)
    cos, sin = tables(30, 64, device)
    for where, kw in (((kp, vp, s.table, s.lens), dict(k_scales=ks, v_scales=vs)),
                      ((s.k_pages, s.v_pages, s.table[:, :0], s.lens), s.kw)):
        assert not ako.paged_attention(s.q, *where, **kw).any()
        assert ako.rope_qk_paged(s.q, s.k, s.v, cos, sin, *where, **kw).isnan().all()
        assert not any(t.any() for t in ako.paged_read(*where, 4, torch.float16, **kw))
    none = torch.empty(0, 32, device=device)  # positions without a table row
    assert ako.rope_qk_paged(s.q, s.k, s.v, none, none, *s.where, **s.kw).isnan().all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("news", [1, 40])
def test_views(news: int, device: str) -> None:
    """Query rows that are one row, a table that is part of a wider one, scales of tokens-major pages."""
    s = step([100, 70], [news, news], heads=8, dtype=torch.float16, device=device)
    whole = s.q
    s.q = whole[:, :, :1].expand(-1, -1, 8, -1)
    check(s)
    s.q = whole[:, :1].expand(-1, news, -1, -1)
    check(s)
    s = step([100, 70], [news, news], head_dim=80, dtype=torch.bfloat16, mx=True, device=device)
    wide = torch.full((2, s.table.shape[1] + 5), -7, dtype=torch.int32, device=device)
    wide[:, 2:-3] = s.table
    s.table = wide[:, 2:-3]
    s.k_scales, s.v_scales = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (s.k_scales, s.v_scales))
    check(s)


@pytest.mark.parametrize("device", DEVICES)
def test_many_heads_on_one_key_head_and_large_pages(device: str) -> None:
    for heads, kv_heads in ((130, 1), (51, 3)):
        for news in (1, 3):
            check(step([90, 40], [news, news], heads=heads, kv_heads=kv_heads, dtype=torch.bfloat16, device=device))
    for page in (300, 1024):
        for mx in (False, True):
            check(step([700, 35], [30, 30], dtype=torch.float16, mx=mx, page=page, device=device))

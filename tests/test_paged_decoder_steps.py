"""Steps of the decoder on a paged cache that fail."""

from __future__ import annotations

import pytest
import torch

from ako_amd.models.decoder import ModelConfig, build_stack

SIZES = dict(hidden_dim=64, n_layers=3, n_heads=4, n_kv_heads=2, intermediate_dim=96, max_seq_len=32, vocab_size=50, eps=1e-6)
gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("wrong", ["batch", "layers", "width", "type", "interrupt"])
def test_a_step_that_fails_leaves_the_cache_where_it_was(wrong: str, device: str, monkeypatch) -> None:
    """Refused before the first layer, or ended in a later one: the lengths are those from before, and the
    next step's result is that of a cache that has not seen the failed one."""
    model = build_stack(ModelConfig(**SIZES), seed=3, device=device)
    x = torch.randn(2, 9, 64, generator=torch.Generator().manual_seed(1)).to(device)
    new = lambda: model.new_paged_cache(16, batch=2, page_size=4)  # noqa: E731
    with torch.no_grad():
        untouched, cache = new(), new()
        model(x[:, :5], kv_cache=untouched)
        model(x[:, :5], kv_cache=cache)
        bad, raised = {"batch": (x[:1, :3], ValueError), "layers": (x[:, :3] + 1, IndexError), "width": (x[:, :3, :32], Exception),
                       "type": (x[:, :3].double(), Exception), "interrupt": (x[:, :3] - 1, KeyboardInterrupt)}[wrong]
        with monkeypatch.context() as m:
            if wrong == "layers":
                m.setattr(cache, "pools", cache.pools[:2])
            if wrong == "interrupt":
                def stop(*a, **k):
                    raise KeyboardInterrupt
                m.setattr(model.layers[1].mlp, "forward", stop)
            with pytest.raises(raised):
                model(bad, kv_cache=cache)
        assert cache.length == 5 and cache.seq_lens.tolist() == [5, 5]
        assert torch.equal(model(x[:, 5:], kv_cache=cache), model(x[:, 5:], kv_cache=untouched))
    assert cache.length == untouched.length == 9 and cache.seq_lens.tolist() == [9, 9]

"""Steps of the decoder on a paged cache that fail, and what a captured step keeps alive."""

from __future__ import annotations

import contextlib
import gc
import weakref

import pytest
import torch

from ako_amd.models.decoder import GraphedGreedy, ModelConfig, build_lm, build_stack

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


def longer_cache(model):
    """A forward on a cache longer than the model's own limit: the stack then needs longer tables."""
    with torch.no_grad():
        model.logits_last(torch.zeros(1, 2, dtype=torch.long, device=model.embed.weight.device),
                          model.stack.new_paged_cache(200, page_size=16))
    gc.collect()


@pytest.mark.parametrize("paged", [False, True])
def test_the_tables_that_a_graph_reads_live_as_long_as_its_runner(paged: bool, monkeypatch) -> None:
    """On a CPU, with capture and replay replaced by nothing: whose memory is kept."""
    class Stub:
        def wait_stream(self, other) -> None: ...
        def replay(self) -> None: ...

    for name, value in (("Stream", Stub), ("current_stream", Stub), ("CUDAGraph", Stub), ("synchronize", lambda: None),
                        ("stream", lambda s: contextlib.nullcontext()), ("graph", lambda g: contextlib.nullcontext())):
        monkeypatch.setattr(torch.cuda, name, value)
    model = build_lm(ModelConfig(**SIZES), dtype=torch.float32, seed=5)
    prompt = torch.randint(0, 50, (1, 7), generator=torch.Generator().manual_seed(0))
    with torch.no_grad():
        runner = GraphedGreedy(model, prompt, 6, cache=model.stack.new_paged_cache(13) if paged else None)
    tables = [weakref.ref(t) for t in model.stack._rope_tables]
    longer_cache(model)
    assert model.stack._rope_tables[0].shape[0] >= 200  # others by now
    assert all(t() is not None and t().shape[0] == 32 for t in tables)
    del runner
    gc.collect()
    assert all(t() is None for t in tables)


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")
@pytest.mark.parametrize("paged", [False, True])
def test_a_replay_after_longer_tables_were_built(paged: bool) -> None:
    prompt = torch.randint(0, 50, (1, 9), generator=torch.Generator().manual_seed(0)).cuda()
    model = build_lm(ModelConfig(**SIZES), dtype=torch.float16, seed=5, device="cuda", init_std=0.2)
    with torch.no_grad():
        new = lambda: model.stack.new_paged_cache(20, page_size=16) if paged else None  # noqa: E731
        want = GraphedGreedy(model, prompt, 10, cache=new()).run().clone()
        runner = GraphedGreedy(model, prompt, 10, cache=new())
        longer_cache(model)
        taken = [torch.full((32, 8), float("nan"), device="cuda") for _ in range(64)]  # what was freed is used again
        assert torch.equal(runner.run(), want)
    del taken


def test_graphed_decoding_refuses_a_cache_of_several_sequences() -> None:
    model = build_lm(ModelConfig(**SIZES), dtype=torch.float32, seed=5)
    cache = model.stack.new_paged_cache(20, batch=2)
    with torch.no_grad(), pytest.raises(ValueError, match="empty cache of 15 positions and one sequence"):
        GraphedGreedy(model, torch.zeros(1, 9, dtype=torch.long), 6, cache=cache)
    assert cache.length == 0 and not cache.seq_lens.any()

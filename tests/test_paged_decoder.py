"""The decoder on a paged cache: prompts in one piece and in chunks, decoding, 8-bit pages, windows,
and every step replayed from a graph."""

from __future__ import annotations

import pytest
import torch

from ako_amd.models.decoder import GraphedGreedy, ModelConfig, build_lm, build_stack
from ako_amd.validation.numerical import assert_close

CFG = ModelConfig(hidden_dim=64, n_layers=2, n_heads=4, n_kv_heads=2, intermediate_dim=96, max_seq_len=64,
                  vocab_size=50, eps=1e-6)
gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]


@pytest.mark.parametrize("device", DEVICES)
def test_chunks_and_steps_match_one_pass(device: str) -> None:
    model = build_stack(CFG, seed=3, device=device)
    x = torch.randn(3, 24, 64, generator=torch.Generator().manual_seed(1)).to(device)
    with torch.no_grad():
        whole = model(x)
        cache = model.new_paged_cache(40, batch=3, page_size=7)
        parts = [model(x[:, a:b], kv_cache=cache) for a, b in ((0, 9), (9, 10), (10, 21), (21, 22), (22, 24))]
    assert cache.length == 24 and cache.seq_lens.tolist() == [24] * 3
    assert_close(torch.cat(parts, 1), whole, atol=1e-4, rtol=1e-4)
    k, v = cache.read(1)
    assert k.shape == v.shape == (3, 24, 2, 16) and bool(k.abs().sum(-1).all())


@pytest.mark.parametrize("device", DEVICES)
def test_windows_forget_and_sinks_stay(device: str) -> None:
    """With a window, a token that left every layer's reach no longer matters; one among the sinks does."""
    one = ModelConfig(hidden_dim=64, n_layers=1, n_heads=4, n_kv_heads=2, intermediate_dim=96, max_seq_len=64, eps=1e-6)
    model = build_stack(one, seed=4, device=device)
    x = torch.randn(1, 20, 64, generator=torch.Generator().manual_seed(2)).to(device)
    outs = {}
    for name, at in (("none", None), ("sink", 1), ("middle", 8)):
        y = x.clone()
        if at is not None:
            y[:, at] += 1.0
        with torch.no_grad():
            outs[name] = model(y, kv_cache=model.new_paged_cache(32, page_size=4, window=5, sinks=2))[:, -1]
    assert torch.equal(outs["none"], outs["middle"]) and not torch.allclose(outs["none"], outs["sink"])


@pytest.mark.parametrize("device", DEVICES)
def test_quantised_pages_hold_what_was_written(device: str) -> None:
    model = build_stack(CFG, seed=5, device=device)
    x = torch.randn(2, 12, 64, generator=torch.Generator().manual_seed(3)).to(device)
    with torch.no_grad():
        plain, small = model.new_paged_cache(16, batch=2), model.new_paged_cache(16, batch=2, quantized=True)
        model(x, kv_cache=plain)
        model(x, kv_cache=small)
    for a, b in zip(plain.read(0), small.read(0, torch.float32)):  # the first layer's are the same but for the format
        largest = a.abs().amax(-1, keepdim=True)  # half a step of e4m3: 2^-4 of a value, or of the block's scale times 2^-6
        assert ((a - b).abs() <= torch.maximum(a.abs() * 2 ** -4, largest * 2.0 ** -16)).all()


def test_limits() -> None:
    model = build_stack(CFG, seed=6)
    cache = model.new_paged_cache(5, page_size=4)
    x = torch.randn(1, 6, 64)
    with torch.no_grad():
        with pytest.raises(ValueError, match="overflow"):
            model(x, kv_cache=cache)
        assert cache.length == 0 and int(cache.seq_lens) == 0
        model(x[:, :5], kv_cache=cache)
        with pytest.raises(ValueError, match="overflow"):
            model(x[:, :1], kv_cache=cache)
        cache.rewind(2)
        model(x[:, :1], kv_cache=cache)
        assert cache.length == 4
        with pytest.raises(ValueError, match="rewind"):
            cache.rewind(5)
        with pytest.raises(ValueError, match="backend"):
            build_stack(CFG, backend="torch", seed=6)(x, kv_cache=model.new_paged_cache(8))


def test_greedy_generation_matches_the_dense_cache() -> None:
    prompt = torch.randint(0, 50, (1, 7), generator=torch.Generator().manual_seed(0))
    model = build_lm(CFG, dtype=torch.float32, seed=5)
    a = model.generate_greedy(prompt, 6)
    assert torch.equal(a, model.generate_greedy(prompt, 6, kv_cache=model.stack.new_paged_cache(13, page_size=4)))


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")
@pytest.mark.parametrize("quantized", [False, True])
def test_graph_replays_match_eager_steps(quantized: bool) -> None:
    prompt = torch.randint(0, 50, (1, 21), generator=torch.Generator().manual_seed(0)).cuda()
    model = build_lm(CFG, dtype=torch.float16, seed=5, device="cuda", init_std=0.2)
    with torch.no_grad():
        new = lambda: model.stack.new_paged_cache(40, page_size=16, quantized=quantized, window=12, sinks=2)  # noqa: E731
        eager = model.generate_greedy(prompt, 16, kv_cache=new())
        model.config.max_seq_len = 64
        runner = GraphedGreedy(model, prompt, 16, cache=new())
        assert torch.equal(runner.run(), eager)
        with pytest.raises(ValueError, match="empty cache"):
            GraphedGreedy(model, prompt, 30, cache=new())


def test_the_benchmark_decodes_on_the_cache_it_is_asked_for(monkeypatch) -> None:
    """``run_config5`` on a CPU stub of the graph runner: which cache each choice hands to it."""
    from ako_amd.models import bench_decoder

    seen = []

    class Runner:
        def __init__(self, model, prompt, steps, *, cache=None):
            seen.append(cache)
            self.steps = steps

        def run(self):
            return torch.zeros(1, self.steps, dtype=torch.long)

    monkeypatch.setattr(bench_decoder, "GraphedGreedy", Runner)
    monkeypatch.setattr(bench_decoder, "config5", lambda: ModelConfig(**{**CFG.__dict__}))
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    for choice, dtype in (("static", None), ("paged", torch.float16), ("paged-mx8", torch.float8_e4m3fn)):
        seen.clear()
        out = bench_decoder.run_config5("ako", prompt_len=5, decode_steps=3, repeats=1, device="cpu", prefill_warmup=0,
                                        prefill_repeats=1, graph_cache=choice)
        assert (seen[0] is None) == (choice == "static") and ("graphed_cache" in out) == (choice != "static")
        if dtype is not None:
            assert seen[0].pools[0][0].dtype == dtype and seen[0].max_len == 8

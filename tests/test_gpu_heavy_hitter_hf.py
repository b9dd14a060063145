"""The heavy-hitter technique end to end: a small Qwen2 (bf16 and fp16, head dim 64, GQA 2) whose layers hold at most 48
tokens per head. Every attention call of the run (the prompt's, each step's) is checked against the 64-bit oracle on the
queries, keys and values it was given and the cache it found, and what the caches hold against the tokens seen."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from budget_cases import assert_output, f64, score_error
from oracle import budget as ob
from test_gpu_eviction import states
from test_gpu_hf import prompt, tiny_model

pytestmark = pytest.mark.gpu

BUDGET, RECENT, FIRST = 48, 8, 2


def config(**more):
    from economize_amd.techniques import HeavyHitterConfig

    return HeavyHitterConfig(budget=BUDGET, recent=RECENT, first=FIRST, **more)


@pytest.fixture
def checked(monkeypatch):
    """The layers' calls, each checked as it returns."""
    from economize_amd import hf

    calls = {"prompt": 0, "mass": 0, "evict": 0, "step": 0}
    prompt_attention, attention_mass = hf.prompt_attention, hf.attention_mass
    evict_prompt, heavy_hitter_attention = hf.evict_prompt, hf.heavy_hitter_attention

    def bounds(rows):
        return tuple(x.cpu().numpy() for x in rows)

    def on_prompt(q, k, v, rows, n, scale, *, softcap, sinks, return_lse):
        out, lse = prompt_attention(q, k, v, rows, n, scale, softcap=softcap, sinks=sinks, return_lse=return_lse)
        want, want_lse, size = ob.prompt_attention(f64(q), f64(k), f64(v), bounds(rows), bounds(rows), scale, softcap)
        assert_output(out, want, size, score_error(q, k, scale, n))
        calls["prompt"] += 1
        return out, lse

    def on_mass(q, k, lse, rows, n, scale, *, window, softcap):
        mass = attention_mass(q, k, lse, rows, n, scale, window=window, softcap=softcap)
        want = ob.attention_mass(f64(q), f64(k), f64(lse), bounds(rows), bounds(rows), scale, softcap, window)
        error = score_error(q, k, scale, n) + (2 * n / 32 + 32) * 2.0 ** -24
        assert (np.abs(f64(mass) - want) <= error * 1.01 * want + 1e-30).all()
        calls["mass"] += 1
        return mass

    def on_evict(cache, k, v, mass, rows, n):
        evict_prompt(cache, k, v, mass, rows, n)
        for b, (lo, hi) in enumerate(zip(*(x.tolist() for x in rows))):
            for h in range(k.shape[1]):
                kept = ob.evict(f64(mass[h, lo:hi]), cache.budget, RECENT, FIRST)
                assert cache.position[b, h, : len(kept)].tolist() == kept.tolist()
                assert torch.equal(cache.keys[b, h, : len(kept)], k[torch.from_numpy(lo + kept).cuda(), h])
        calls["evict"] += 1

    def on_step(cache, q, k, v, scale, softcap, sinks, out):
        before = states(cache)
        heavy_hitter_attention(cache, q, k, v, scale, softcap, sinks, out=out)
        error = score_error(q, torch.cat([k[:, :, None], cache.keys], 2), scale, cache.budget)
        after = states(cache)
        for b, state in enumerate(before):
            want, size = ob.heavy_step(state, f64(q[b]), f64(k[b]), f64(v[b]), cache.budget, RECENT, FIRST,
                                       scale)
            assert_output(out[b], want, size, error)
            assert np.array_equal(after[b]["position"], state["position"])
            assert np.array_equal(after[b]["keys"], state["keys"])
        calls["step"] += 1
        return out

    for name, fn in (("prompt_attention", on_prompt), ("attention_mass", on_mass), ("evict_prompt", on_evict),
                     ("heavy_hitter_attention", on_step)):
        monkeypatch.setattr(hf, name, fn)
    return calls


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window", [None, 16])
def test_generate(checked, dtype, window) -> None:
    from economize_amd.attention import kernel_usage
    from economize_amd.hf import HeavyHitterLayer, apply

    em = apply(tiny_model("sdpa", dtype), config(window=window, layers=(1, 2, 4)))
    kernel_usage(reset=True)
    ids = prompt()
    cache = em.make_cache(200)
    with torch.no_grad():
        logits = em.model(input_ids=ids, past_key_values=cache, use_cache=True).logits
        for _ in range(20):
            token = logits[:, -1].argmax(-1, keepdim=True)
            logits = em.model(input_ids=token, past_key_values=cache, use_cache=True).logits
            assert torch.isfinite(logits).all()
    assert checked == {"prompt": 3, "mass": 3, "evict": 3, "step": 60}
    for layer in cache.layers:
        if isinstance(layer, HeavyHitterLayer):
            c = layer.cache
            assert layer.get_seq_length() == 90 and c.length.tolist() == [90] and (c.count == BUDGET).all()
            for h in range(2):
                held = sorted(c.position[0, h].tolist())
                assert len(set(held)) == BUDGET and held[:FIRST] == list(range(FIRST))
                assert held[-RECENT:] == list(range(90 - RECENT, 90))
    paths = {(r["layer"], r["path"]) for r in kernel_usage()}
    assert all((i, "kernel_heavy_hitter") in paths for i in (0, 1, 3))
    out = em.generate(ids, 8)
    assert out.shape == (1, ids.shape[1] + 8)


def test_a_budget_larger_than_the_text_keeps_every_token(checked) -> None:
    """Nothing is evicted, so the prompt's K/V are held as they were written, in order."""
    from economize_amd import hf
    from economize_amd.techniques import HeavyHitterConfig

    em = hf.apply(tiny_model("sdpa"), HeavyHitterConfig(budget=256, recent=8, first=2))
    cache = em.make_cache(200)
    with torch.no_grad():
        em.model(input_ids=prompt(), past_key_values=cache, use_cache=True)
        em.model(input_ids=prompt()[:, :5], past_key_values=cache, use_cache=True)  # several tokens in one pass
    for layer in cache.layers:
        assert layer.cache.position[0, :, :75].tolist() == [list(range(75))] * 2
        assert layer.cache.count.tolist() == [[75, 75]]
    assert checked["step"] == 20


def test_left_padded_batch(checked) -> None:
    from economize_amd.hf import apply

    em = apply(tiny_model("sdpa"), config())
    ids = prompt().repeat(3, 1)
    mask = torch.ones_like(ids)
    mask[1, :25] = 0
    mask[2, :69] = 0
    cache = em.make_cache(200)
    with torch.no_grad():
        logits = em.model(input_ids=ids, attention_mask=mask, past_key_values=cache, use_cache=True).logits
        for _ in range(6):
            mask = torch.cat([mask, mask.new_ones(3, 1)], 1)
            token = logits[:, -1].argmax(-1, keepdim=True)
            logits = em.model(input_ids=token, attention_mask=mask, past_key_values=cache, use_cache=True).logits
            assert torch.isfinite(logits).all()
    for layer in cache.layers:
        assert layer.cache.length.tolist() == [76, 51, 7]
        assert layer.cache.count.tolist() == [[48, 48], [48, 48], [7, 7]]


def test_other_masks_and_weights_are_refused() -> None:
    from economize_amd.errors import ConfigError
    from economize_amd.hf import apply

    em = apply(tiny_model("sdpa"), config())
    ids = prompt().repeat(2, 1)
    hole = torch.ones_like(ids)
    hole[0, 30] = 0
    with pytest.raises(ConfigError, match="causal mask of a left-padded or full batch"), torch.no_grad():
        em.model(input_ids=ids, attention_mask=hole, past_key_values=em.make_cache(200), use_cache=True)
    cache = em.make_cache(200)
    padded = torch.ones_like(ids)
    padded[0, :9] = 0
    with torch.no_grad():
        em.model(input_ids=ids, attention_mask=padded, past_key_values=cache, use_cache=True)
        with pytest.raises(ConfigError, match="needs its mask in every pass"):
            em.model(input_ids=ids[:, :1], past_key_values=cache, use_cache=True)


def test_captured_step() -> None:
    """A layer's step, update and attention together, captured and replayed with new tokens: equal to an eager twin."""
    from economize_amd.attention import economize_attention_forward
    from economize_amd.hf import HeavyHitterLayer

    gen = torch.Generator().manual_seed(3)

    def tokens(t):
        return tuple(torch.randn(2, h, t, 64, generator=gen).to(torch.bfloat16).cuda() for h in (4, 2, 2))

    layers = [HeavyHitterLayer(config()) for _ in range(2)]

    def run(layer, q, k, v):
        keys, values = layer.update(k, v)
        return economize_attention_forward(None, q, keys, values, None)[0]

    p = tokens(70)
    for layer in layers:
        run(layer, *p)
    new = tokens(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(layers[0], *new)
    torch.cuda.synchronize()
    run(layers[1], *new)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = run(layers[0], *new)
    for i in range(6):
        for a, b in zip(new, tokens(1)):
            a.copy_(b)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, run(layers[1], *new)), i
        torch.cuda.synchronize()
        for name in ("keys", "values", "score", "position", "count", "length"):
            assert torch.equal(getattr(layers[0].cache, name), getattr(layers[1].cache, name)), (i, name)


def test_reordered_rows() -> None:
    from economize_amd.hf import HeavyHitterLayer

    layer = HeavyHitterLayer(config())
    k = torch.randn(2, 2, 5, 64, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
    layer.lazy_initialization(k, k)
    layer.cache.keys[:, :, :5] = k
    layer.reorder_cache(torch.tensor([1, 1]))
    assert torch.equal(layer.cache.keys[0, :, :5], k[1]) and torch.equal(layer.cache.keys[1, :, :5], k[1])
    layer.cache.check()

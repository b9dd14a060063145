"""The heavy-hitter technique's configuration, validation and layer bookkeeping on the CPU."""

from __future__ import annotations

import json

import pytest
import torch

from economize_amd.attention import accepts_packed_kv
from economize_amd.errors import ConfigError, IncompatibleTechniquesError
from economize_amd.techniques import HeavyHitterConfig, HeavyHitterTechnique, QuestConfig, technique_for
from test_hf import tiny_model


def test_config() -> None:
    for fields, match in (({"budget": 0}, "budget"), ({"recent": 0}, "recent"), ({"first": -1}, "first"),
                          ({"first": True}, "first"), ({"budget": 100, "recent": 97}, "exceed the budget"),
                          ({"window": 0}, "window"), ({"layers": [1]}, "tuple")):
        with pytest.raises(ConfigError, match=match):
            HeavyHitterConfig(**fields)
    config = HeavyHitterConfig(budget=256, window=32, layers=(2, 3))
    assert HeavyHitterConfig.from_dict(json.loads(json.dumps(config.to_dict()))) == config
    technique = technique_for(config)
    assert isinstance(technique, HeavyHitterTechnique) and technique.covers(2) and not technique.covers(1)
    cache = technique.make_cache(batch=3, kv_heads=2, head_dim=64, device="cpu", dtype=torch.float16)
    assert cache.budget == 256 and cache.keys.shape == (3, 2, 256, 64)


def test_validate() -> None:
    assert accepts_packed_kv("economize", "heavy_hitter")
    config = HeavyHitterConfig()
    config.validate(tiny_model(attn="economize").to(torch.bfloat16))
    with pytest.raises(ConfigError, match="head dims"):
        config.validate(tiny_model(head_dim=32, attn="economize").to(torch.bfloat16))
    with pytest.raises(ConfigError, match="bf16 and fp16"):
        config.validate(tiny_model(attn="economize"))
    with pytest.raises(IncompatibleTechniquesError, match="heavy-hitter cache"):
        config.validate(tiny_model().to(torch.bfloat16))


def test_apply_and_caches() -> None:
    from economize_amd.hf import HeavyHitterLayer, apply

    model = tiny_model().to(torch.bfloat16)
    with pytest.raises(IncompatibleTechniquesError, match="one KV technique per layer"):
        apply(model, HeavyHitterConfig(), QuestConfig())
    em = apply(model, HeavyHitterConfig(layers=(3, 4)), QuestConfig(layers=(2,), dense_layers=0))
    cache = em.make_cache(64)
    assert [isinstance(x, HeavyHitterLayer) for x in cache.layers] == [False, False, True, True]
    with pytest.raises(ConfigError, match="static cache"):
        em.make_cache(64, static=True)


def test_a_pass_nothing_attended_over_is_an_error() -> None:
    from economize_amd.hf import HeavyHitterLayer

    layer = HeavyHitterLayer(HeavyHitterConfig(budget=8, recent=2, first=1), layer=5)
    k = torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16)
    keys, _ = layer.update(k, k)
    assert torch.equal(keys, k) and layer.get_seq_length() == 3
    with pytest.raises(IncompatibleTechniquesError, match="layer 5 was not attended over"):
        layer.update(k, k)
    layer.reset()
    assert layer.get_seq_length() == 0
    keys, _ = layer.update(k, k)
    from economize_amd.attention import economize_attention_forward

    with pytest.raises(ConfigError, match="cannot fall back \\(cpu\\)"):
        economize_attention_forward(None, torch.zeros(1, 4, 3, 64, dtype=torch.bfloat16), keys, k, None)

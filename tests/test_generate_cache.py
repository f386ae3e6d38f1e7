"""The cache that generate keeps between calls, and how much of it a call asks for (no GPU)."""
import weakref

import pytest
import torch

import tiny_models as tm

import pytorch_transformers_b200 as ptb


@pytest.fixture
def model():
    config = tm.config_dict("A")
    return ptb.AutoModelForCausalLM.from_config(ptb.FalconConfig.from_dict(config), seed=1, dtype="bfloat16", device="cpu")


@pytest.mark.parametrize("asked", [(640, None), (64, torch.float8_e4m3fn), (640, torch.float8_e4m3fn)])
def test_the_old_cache_is_gone_before_the_next_is_allocated(model, monkeypatch, asked):
    old = weakref.ref(model._ensure_cache(320))
    assert model._ensure_cache(128) is old()
    seen = []
    make = model.new_cache

    def new_cache(*args, **kwargs):
        seen.append(old() is None)
        return make(*args, **kwargs)
    monkeypatch.setattr(model, "new_cache", new_cache)
    cache = model._ensure_cache(*asked)
    assert seen == [True] and cache.max_tokens >= asked[0] and cache.kv_dtype == asked[1]


def test_a_cache_with_open_sequences_is_left_to_its_holder(model):
    cache = model._ensure_cache(320)
    slot = cache.open()
    assert model._ensure_cache(64) is not cache
    assert slot in cache.records

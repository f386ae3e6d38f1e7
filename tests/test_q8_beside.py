"""Steps over a cache in 8 bits beside the feed-forward's weight stream: when, and how many blocks the attention takes from it."""
import types

import pytest
import torch

import tiny_models as tm

import pytorch_transformers_b200 as ptb
from pytorch_transformers_b200 import kernels as K


def attention():
    config = ptb.FalconConfig.from_dict(tm.config_dict("A"))
    model = ptb.AutoModelForCausalLM.from_config(config, seed=1, dtype="bfloat16", device="cpu")
    return model._mixers[0], model


@pytest.mark.parametrize("keys", [1, 1000, 100_000, 160_000, 200_000, 320_000, 330_000, 10 ** 7])
def test_a_step_runs_beside_the_stream_over_either_cache(keys):
    # 40 MB of bfloat16 keys and values is where it stops; in 8 bits the same keys
    mixer, model = attention()
    answers = []
    for kv_dtype in (None, torch.float8_e4m3fn):
        cache = model.new_cache(64, kv_dtype=kv_dtype)
        ctx = types.SimpleNamespace(past=[keys - 1], new=[1], cache=cache)
        answers.append(mixer.runs_beside(ctx))
    assert answers[0] == answers[1] == (keys * mixer.kv_heads * mixer.head_dim * 4 <= K.DECODE_BESIDE_MAX_KV_BYTES)


@pytest.mark.parametrize("side", [None, object()])
def test_the_attention_is_told_of_the_stream(side, monkeypatch):
    mixer, model = attention()
    seen = []
    monkeypatch.setattr(mixer.build.kernels, "attention_decode_q8", lambda *a, **kw: seen.append(kw["beside"]))
    ctx = types.SimpleNamespace(past=[5], new=[1], pages_hint=1, side_stream=side)
    tiles = types.SimpleNamespace(facts={"mma_tokens": 1})
    mixer._attend_q8(None, (None,) * 4, ctx, types.SimpleNamespace(writes_cache=True), tiles, None, None, None, False)
    assert seen == [side is not None]


@pytest.mark.gpu
@pytest.mark.parametrize("kv,rows,dim", [(1, 71, 64), (8, 4, 128), (2, 1, 256), (8, 16, 64)])
@pytest.mark.parametrize("seqs", [1, 2, 3, 8, 16, 64])
@pytest.mark.parametrize("pages", [1, 3, 33, 300, 5000])
def test_half_of_the_device_is_the_streams(kv, rows, dim, seqs, pages):
    L, sms = K.lib(), K.sm_count("cuda")
    splits = L.ptb_attention_decode_q8_splits_beside(seqs, kv, rows, dim, pages)
    assert splits in (1, 2, 4) or splits % 8 == 0
    assert splits == 1 or (splits * seqs * kv <= sms // 2 and splits <= pages // 2)


@pytest.mark.gpu
def test_the_result_beside_a_stream():
    from test_q8_gpu import Case
    c = Case(1, 71, 64, [900, 2000, 5], [1, 1, 1], rot=64, seed=2)
    cache, batch = c.device(K)
    for beside in (False, True):
        keep = [t.clone() for t in cache]
        out = K.attention_decode_q8(c.dev["fused"], *keep, batch, c.dev["rope"], None, 1, 71, 64, c.scale, beside=beside)
        if not beside:
            c.append()
        c.check(out, c.split()[0])
    K.check_device_errors("cuda")

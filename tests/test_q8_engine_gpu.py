"""The cache in 8 bits and its page operations under the engine: the attention part on a step, models through step and generate,
sequences forked, cut and moved between steps."""
import pytest
import torch

import plain_q8 as plain
import tiny_models as tm
from cache_pages_model import Sequences, random_walk

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn
BF = torch.bfloat16


@pytest.mark.parametrize("seed", range(3))
@pytest.mark.parametrize("kw", [dict(), dict(window=100, dtype=BF), dict(state=3), dict(dtype=BF, kv_dtype=F8)], ids=str)
def test_random_walks_of_the_cache(seed, kw):
    random_walk(Sequences("cuda", **kw), seed, 40)


def identity_part(kv, qpk, dim, position, window):
    """An attention part whose projection passes its input on and whose output projection passes the heads on."""
    from pytorch_transformers_b200 import kernels as K
    from pytorch_transformers_b200.parts import BuildContext, PartSpec
    from pytorch_transformers_b200.parts.base import make_part
    width = kv * (qpk + 2) * dim
    children = {"rotary": {"position": PartSpec("position", "rotary", dict(head_dim=dim, theta=10000.0))},
                "alibi": {"position": PartSpec("position", "alibi", dict(heads=kv * qpk))}, "none": {}}[position]
    part = make_part(BuildContext(torch.device("cuda"), BF, K),
                     PartSpec("mixer", "attention", dict(hidden=width, heads=kv * qpk, kv_heads=kv, head_dim=dim, window=window), children=children))
    part.bind({"qkv.weight": torch.eye(width, dtype=BF, device="cuda"),
               "out.weight": torch.eye(kv * qpk * dim, dtype=BF, device="cuda")})
    return part


@pytest.mark.parametrize("kv,qpk,dim", [(1, 71, 64), (2, 4, 128), (2, 3, 48), (1, 130, 16)])
@pytest.mark.parametrize("position,window", [("rotary", 0), ("alibi", 0), ("none", 50)])
@pytest.mark.parametrize("new", [[1, 1, 1], [5, 16, 1], [40, 2, 64], [200, 1, 130]])
def test_attention_part(kv, qpk, dim, position, window, new):
    from pytorch_transformers_b200.cache import Cache
    from pytorch_transformers_b200.engine.batch import StepContext
    from pytorch_transformers_b200.parts import ScheduleEntry
    part = identity_part(kv, qpk, dim, position, window)
    cache = Cache([(0, part.cache_need(), None)], 64 * 24, BF, "cuda", kv_dtype=F8)
    g = torch.Generator().manual_seed(dim)
    slots, pasts = [cache.open() for _ in new], [100, 3, 64]
    for counts in (pasts, new):
        x = torch.randn(sum(counts), kv * (qpk + 2) * dim, generator=g).to(BF)
        past = [cache.length(s) for s in slots]
        ctx = StepContext(cache, slots, [[0] * n for n in counts], 1, [[] for _ in new], [part.planner()])
        out = part.forward(x.cuda(), ctx, ScheduleEntry(0, 0))
        part.build.kernels.check_device_errors("cuda")
        tables = [list(cache.pages(s, 0)) for s in slots]
        ctx.commit()
    cos = sin = None
    if position == "rotary":
        cos, sin = (t.cpu() for t in part.build.kernels.rope_table(ctx.dev["tok_pos"], part.position.rotation()))
    f = x.float().view(-1, kv, qpk + 2, dim)
    q = plain.rotate(f[:, :, :qpk].reshape(-1, kv * qpk, dim), cos, sin, False)
    # the step's keys and values are in the pages as codes: those are what it attends over
    grp = cache.groups[0]
    at = 0
    for b, (n, p) in enumerate(zip(new, past)):
        ids = torch.tensor(tables[b]).clamp(min=0)
        k, v = (plain.values(c[0].float().cpu().double(), e[0].cpu())[ids].transpose(1, 2).reshape(-1, kv, dim)[:p + n]
                for c, e in ((grp.k, grp.k_exp), (grp.v, grp.v_exp)))
        slopes = part.position.score_bias().cpu() if position == "alibi" else None
        want, most, size = plain.attend(q[at:at + n], k, v, part.scale, torch.arange(p, p + n), slopes, window)
        # prompts' queries are bfloat16 numbers (8 bits), and long ones with slopes have weights of 8 bits
        limit = plain.bound(want, most, size, p + n, q_bits=11 if max(new) == 1 else 8, weight_bits=7)
        got = out[at:at + n].double().cpu().view(want.shape)
        assert bool(((got - want).abs() <= limit).all())
        at += n


def model_of(tmp_path, name="E", dtype="bfloat16"):
    import pytorch_transformers_b200 as ptb
    return ptb.AutoModelForCausalLM.from_pretrained(tm.tiny_folder(str(tmp_path), name, bf16=dtype == "bfloat16"), dtype=dtype)


@pytest.mark.parametrize("name", ["A", "D", "E", "F", "G"])
def test_steps_in_8_bits_replayed_and_not(tmp_path, name, monkeypatch):
    from pytorch_transformers_b200 import kernels as K
    model = model_of(tmp_path, name)
    # a replayed step's page tables come in whole buckets, and how many blocks share a sequence's pages follows from their width; with
    # the same number of blocks both form the same sums in the same order
    decode = K.attention_decode_q8
    monkeypatch.setattr(K, "attention_decode_q8", lambda *a, **kw: decode(*a, n_splits=2, **kw))
    prompts = tm.prompts(name, (70, 5, 130), seed=2)
    runs = []
    for graphs in (False, True):
        model.use_graphs = graphs
        cache = model.new_cache(64 * 12, kv_dtype=F8)
        slots = [cache.open() for _ in prompts]
        out = [model.step(cache, slots, prompts)]
        out += [model.step(cache, slots, [[t], [t + 1], [t + 2]]) for t in range(3, 73)]
        model.check_errors()
        runs.append(torch.stack(out))
    assert torch.isfinite(runs[0]).all() and torch.equal(runs[0], runs[1])
    # and near the model's own cache: 4 bits of mantissa in keys and values against 8
    cache = model.new_cache(64 * 12)
    slots = [cache.open() for _ in prompts]
    own = [model.step(cache, slots, prompts)] + [model.step(cache, slots, [[t], [t + 1], [t + 2]]) for t in range(3, 73)]
    off = (torch.stack(own) - runs[0]).norm() / torch.stack(own).norm()
    assert 0 < float(off) < 0.25


def test_head_sizes_that_8_bits_do_not_take(tmp_path):
    model = model_of(tmp_path, "B")                   # heads of 12
    with pytest.raises(ValueError, match="8 bits"):
        model.new_cache(640, kv_dtype=F8)
    model = model_of(tmp_path, "A", "float32")
    with pytest.raises(ValueError, match="model's dtype"):
        model.generate([[1, 2]], max_new_tokens=2, cache_dtype="float8_e4m3fn")


def test_generate_in_8_bits(tmp_path):
    model = model_of(tmp_path)
    prompts = tm.prompts("E", (4, 90, 6), seed=3)
    kw = dict(max_new_tokens=8, eos_token_id=None)
    a = model.generate(prompts, cache_dtype="float8_e4m3fn", **kw)
    assert model._cache.kv_dtype == F8 and [len(x) for x in a] == [12, 98, 14]
    assert a == model.generate(prompts, cache_dtype="float8_e4m3fn", **kw)
    model.generate(prompts, **kw)
    assert model._cache.kv_dtype is None


@pytest.mark.parametrize("dtype,kv_dtype", [("float32", None), ("bfloat16", None), ("bfloat16", F8)])
def test_forked_cut_and_moved_between_steps(tmp_path, dtype, kv_dtype):
    model = model_of(tmp_path, dtype=dtype)
    prompt = tm.prompts("E", (150,), seed=5)[0]
    cache = model.new_cache(64 * 16, kv_dtype=kv_dtype)
    a = cache.open()
    model.step(cache, [a], [prompt])
    b = cache.fork(a)
    rows = model.step(cache, [a, b], [[5], [5]])
    assert torch.equal(rows[0], rows[1])              # the same past, the same step
    apart = model.step(cache, [a, b], [[7], [8]])
    assert not torch.equal(apart[0], apart[1])
    # b back to the prompt and on with a's tokens: the same again (in 8 bits the cut-off token's codes are
    # written over; the exponent that it may have raised stays)
    cache.truncate(b, 150)
    model.step(cache, [b], [[5]])
    again = model.step(cache, [b], [[7]])
    if dtype == "float32":
        assert torch.equal(again[0], apart[0])
    else:
        torch.testing.assert_close(again[0], apart[0], atol=5e-2, rtol=5e-2)
    # the pages moved and the storage changed under both
    cache.truncate(b, 152)
    c = cache.fork(a)
    cache.compact()
    cache.check()
    cache.resize(64 * 40)
    moved = model.step(cache, [a, c], [[9], [9]])
    assert torch.equal(moved[0], moved[1])
    fresh = model.new_cache(64 * 16, kv_dtype=kv_dtype)
    s = fresh.open()
    model.step(fresh, [s], [prompt])
    for t in (5, 7):
        model.step(fresh, [s], [[t]])
    want = model.step(fresh, [s], [[9]])
    if dtype == "float32":
        assert torch.equal(moved[0], want[0])
    else:
        torch.testing.assert_close(moved[0], want[0], atol=5e-2, rtol=5e-2)
    model.check_errors()


@pytest.mark.parametrize("max_batch", [64, 2])
def test_shared_prompts_give_the_same_tokens(tmp_path, max_batch):
    model = model_of(tmp_path, dtype="float32")       # rows do not depend on their batch in float32
    prompts = tm.prompts("E", (70, 3), seed=8)
    kw = dict(max_new_tokens=9, do_sample=True, temperature=1.3, seed=4, num_return_sequences=3, eos_token_id=None, max_batch_size=max_batch)
    apart = model.generate(prompts, **kw)
    assert model.generate(prompts, share_prompts=True, **kw) == apart
    assert len({tuple(x) for x in apart}) > 3
    model._cache.check()


def test_a_device_without_a_number_names_the_current_one():
    from pytorch_transformers_b200 import kernels as K
    K.error_flag(torch.device("cuda", torch.cuda.current_device())).fill_(7)
    with pytest.raises(K.KernelError, match="code 7"):
        K.check_device_errors("cuda")
    K.check_device_errors("cuda")

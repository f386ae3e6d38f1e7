"""Attention over a cache in 8 bits against bounds for weights of 11 bits and more, which is what every form of it has."""
import pytest
import torch

import plain_q8 as plain
from test_q8_engine_gpu import F8, identity_part
from test_q8_gpu import BF, PAGE, Case, K, run_prompt  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv,qpk,dim", [(1, 5, 64), (2, 4, 128), (3, 1, 64), (1, 3, 96)])
@pytest.mark.parametrize("window", [0, 200])
@pytest.mark.parametrize("pasts,news", [([0], [129]), ([70, 0, 500], [200, 102, 140]), ([0, 64], [300, 128])])
def test_prompts_with_slopes(K, kv, qpk, dim, pasts, news, window):
    # two terms of 8 bits each, tiles full enough that their pages are unpacked
    c = Case(kv, qpk, dim, pasts, news, slopes=True, window=window, seed=dim + qpk)
    if window:
        c.give_back_left_of_windows()
    out, q = run_prompt(K, c, sum((p + n + PAGE - 1) // PAGE for p, n in zip(pasts, news)), tile=128)
    c.check(out, q)


@pytest.mark.parametrize("kv,qpk,dim", [(1, 71, 64), (2, 4, 128), (2, 3, 48), (1, 130, 16)])
@pytest.mark.parametrize("position,window", [("rotary", 0), ("alibi", 0), ("none", 50)])
@pytest.mark.parametrize("new", [[1, 1, 1], [5, 16, 1], [200, 70, 130]])
def test_attention_part(kv, qpk, dim, position, window, new):
    from pytorch_transformers_b200.cache import Cache
    from pytorch_transformers_b200.engine.batch import StepContext
    from pytorch_transformers_b200.parts import ScheduleEntry
    part = identity_part(kv, qpk, dim, position, window)
    cache = Cache([(0, part.cache_need(), None)], 64 * 24, BF, "cuda", kv_dtype=F8)
    g = torch.Generator().manual_seed(dim)
    slots = [cache.open() for _ in new]
    for counts in ([100, 3, 64], new):
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
    q = plain.rotate(x.float().view(-1, kv, qpk + 2, dim)[:, :, :qpk].reshape(-1, kv * qpk, dim), cos, sin, False)
    grp, at = cache.groups[0], 0
    slopes = part.position.score_bias().cpu() if position == "alibi" else None
    for b, (n, p) in enumerate(zip(new, past)):
        ids = torch.tensor(tables[b]).clamp(min=0)
        k, v = (plain.values(c[0].float().cpu().double(), e[0].cpu())[ids].transpose(1, 2).reshape(-1, kv, dim)[:p + n]
                for c, e in ((grp.k, grp.k_exp), (grp.v, grp.v_exp)))
        want, most, size = plain.attend(q[at:at + n], k, v, part.scale, torch.arange(p, p + n), slopes, window)
        # prompts' queries are bfloat16 numbers (8 bits)
        limit = plain.bound(want, most, size, p + n, q_bits=11 if max(new) == 1 else 8)
        assert bool(((out[at:at + n].double().cpu().view(want.shape) - want).abs() <= limit).all())
        at += n


@pytest.mark.parametrize("kv,qpk,dim,splits", [(1, 1, 64, 0), (2, 20, 128, 1), (1, 3, 256, 1)])
def test_every_step_of_rows_that_raise_exponents(K, kv, qpk, dim, splits):
    # rows that grow by 1.7 a token: each step rounds the earlier codes again and asks for the first pages a second time
    n, width = 70, kv * (qpk + 2) * dim
    c = Case(kv, qpk, dim, [0], [n], seed=3)
    grow = torch.ones(n, kv, qpk + 2, 1)
    grow[:, :, qpk:] = 1.7 ** torch.arange(n)[:, None, None, None]
    whole = (torch.randn(n, kv, qpk + 2, dim, generator=torch.Generator().manual_seed(1)) * grow).view(n, width).to(BF)
    cache, _ = c.device(K)
    table = c.table.cuda()
    for t in range(n):
        step = Case(kv, qpk, dim, [t], [1])
        step.fused, step.table, step.codes, step.exps, step.pages = whole[t:t + 1], c.table, c.codes, c.exps, c.pages
        step.scale = c.scale * 1.7 ** -t      # scores of a few units throughout
        ints = [torch.tensor(x, dtype=torch.int32).cuda() for x in ([0], [t], [0], [1], [t])]
        out = K.attention_decode_q8(step.fused.cuda(), *cache, K.step_batch(*ints, table), None, None, kv, qpk, dim, step.scale, n_splits=splits)
        step.append()
        step.check(out, step.split()[0])
    c.check_cache()
    K.check_device_errors("cuda")

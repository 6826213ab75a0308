"""
The paged-cache operators as a decode loop uses them, through
``RandomLlama.forward_varlen``: prompts of two families enter with a kept page
index, share their prompt pages, then decode with plain attention, with the
shared plan and with the sparse plan.

Both plans compute the plain step's attention (the sparse one when its budget
covers every page) to rounding: per layer an output differs by at most
2 * 2^-11 of its largest value for each of the two paths, which the small
model's residual stream (weights of norm about 1) carries to the logits without
growth beyond a factor of 4 a layer: 2 layers * 4 * 4 * 2^-10 = 2^-5 of the
largest logit. The cached keys of both paths after a step are equal in the
first layer bit for bit.
"""

from __future__ import annotations

import pytest
import torch

from llm_serving_layer_b200 import B200PagedBackend, PageIndex, SharedPrefix, build_meta, sample_greedy
from llm_serving_layer_b200.llama import LlamaConfig, RandomLlama

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
CFG = LlamaConfig(hidden=256, n_layers=2, n_heads=8, n_kv_heads=2, head_dim=64, ffn=512, vocab=1000,
                  rope_positions=2048)


@pytest.fixture(scope="module", autouse=True)
def cuda():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device (run with -m 'not gpu' on CPU)"


def start(validate="host"):
    """Two families of three sequences: 20 shared prompt pages each, then own prompts; the pool after prefill."""
    bk = B200PagedBackend(CFG.n_layers, 160, 16, CFG.n_kv_heads, CFG.n_heads, CFG.head_dim, device=DEV,
                          validate=validate)
    model = RandomLlama(CFG, device=DEV, seed=3, init_std=0.06)
    index = PageIndex(bk)
    ids = torch.randperm(160, generator=torch.Generator().manual_seed(1)).tolist()
    g = torch.Generator(device=DEV).manual_seed(2)
    tables, kv = [], []
    for family in range(2):
        lead = [ids.pop() for _ in range(20)]
        prompt = torch.randint(CFG.vocab, (320,), generator=g, device=DEV)
        model.forward_varlen(prompt, build_meta([lead], [320], [320], 16, device=DEV), bk, index=index)
        for tail in (33, 5, 17):
            own = [ids.pop() for _ in range(4)]
            tables.append(lead + own)
            kv.append(320 + tail)
            more = torch.randint(CFG.vocab, (tail,), generator=g, device=DEV)
            model.forward_varlen(more, build_meta([tables[-1]], [kv[-1]], [tail], 16, device=DEV), bk, index=index)
    return bk, model, index, tables, kv


def test_decode_loop_with_each_plan():
    bk, model, index, tables, kv = start()
    check = PageIndex(bk)  # the index kept while prefilling is the pool's
    done = sorted({t[p] for t, n in zip(tables, kv) for p in range(n // 16)})
    check.rebuild(done)
    assert torch.equal(check.codes[:, done], index.codes[:, done])
    assert torch.equal(check.scales[:, done], index.scales[:, done])
    tokens = torch.arange(6, device=DEV)
    for step in range(18):  # across a page end for some sequences
        kv = [n + 1 for n in kv]
        meta = build_meta(tables, kv, [1] * 6, 16, device=DEV)
        pools = [p.clone() for p in bk.k_pool + bk.v_pool]
        plain = model.forward_varlen(tokens, meta, bk)
        after = [p.clone() for p in bk.k_pool + bk.v_pool]
        shared = bk.plan_shared(meta, SharedPrefix.from_tables(tables, kv, [1] * 6, 16))
        sparse = bk.plan_sparse(meta, index, 24)  # covers every page
        for plan in (dict(shared=shared, index=index), dict(sparse=sparse)):
            for p, was in zip(bk.k_pool + bk.v_pool, pools):
                p.copy_(was)
            got = model.forward_varlen(tokens, meta, bk, **plan)
            bk.check_status()
            assert torch.equal(bk.k_pool[0], after[0]) and torch.equal(bk.v_pool[0], after[2])
            assert float((got - plain).abs().max()) <= 2.0 ** -5 * float(plain.abs().max())
        tokens = sample_greedy(plain)
    few = model.forward_varlen(tokens, build_meta(tables, [n + 1 for n in kv], [1] * 6, 16, device=DEV), bk,
                               sparse=bk.plan_sparse(build_meta(tables, [n + 1 for n in kv], [1] * 6, 16, device=DEV),
                                                     index, 6, sink=1, recent=2))
    bk.check_status()
    assert few.shape == (6, CFG.vocab) and bool(torch.isfinite(few).all())


def test_shared_families_are_found():
    _, _, _, tables, kv = start("device")
    s = SharedPrefix.from_tables(tables, kv, [1] * 6, 16)
    assert s.group_sizes == [3, 3] and s.prefix_pages == [20, 20]


def test_one_plan_a_step():
    bk, model, index, tables, kv = start("device")
    meta = build_meta(tables, kv, [1] * 6, 16, device=DEV)
    with pytest.raises(ValueError, match="not both"):
        model.forward_varlen(torch.zeros(6, dtype=torch.int64), meta, bk,
                             shared=bk.plan_shared(meta, SharedPrefix([6], [0])), sparse=bk.plan_sparse(meta, index, 4))

"""
The paged-cache operators where their inputs are at the edge: tables that are
inconsistent, geometries without the tensor-core kernel, keys and queries that
are not finite, blocks taken over by other writers, pools beyond 4 GiB.

Output bounds are those of ``test_gpu_shared.py`` and ``test_gpu_sparse.py``
(``close``); page lists, index entries and zeros must be equal.
"""

from __future__ import annotations

import dataclasses

import numpy as np
import pytest
import torch

import test_gpu_shared as sh
import test_gpu_sparse as sp
from llm_serving_layer_b200 import B200PagedBackend, PageIndex, SharedPrefix, build_meta
from llm_serving_layer_b200._native import PkvError

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module", autouse=True)
def cuda():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device (run with -m 'not gpu' on CPU)"


def test_a_long_kernel_before_is_waited_for():
    """The kernel before, on one SM, outlasts the limit of the tile role's own waits (1 s): nothing times out."""
    bk, meta, q, shared, tables = sh.build([(21, [(4 + i % 37, 1 + i % 3) for i in range(40)])], validate="device")
    plan = bk.plan_shared(meta, shared)
    want = bk.attend_shared(q, 0, 0.125, plan)
    slow = B200PagedBackend(1, 1, 1024, 1, 1, 64, device=DEV, dtype=torch.float32, validate="device")
    index, one = PageIndex(slow), build_meta([[0]], [1024], [1], 1024, device=DEV)
    x = torch.ones(1, 1, 64, device=DEV)
    at = [torch.cuda.Event(enable_timing=True) for _ in range(2)]

    def run(n, after=lambda: None):  # one row over the same page n times
        splan = slow.plan_sparse(one, index, n, max_pages=1)
        pages = torch.zeros((1, 1, n), dtype=torch.int32, device=DEV)
        at[0].record()
        slow.attend_pages(x, 0, 0.1, splan, pages)
        got = after()
        at[1].record()
        torch.cuda.synchronize()
        return at[0].elapsed_time(at[1]), got

    run(100)
    n = min(40000, int(1600.0 / max(run(100)[0] / 100, 0.04)))
    ms, got = run(n, lambda: bk.attend_shared(q, 0, 0.125, plan))
    assert 1200 < ms < 6000, (ms, n)
    bk.check_status()
    slow.check_status()
    assert torch.equal(got, want)


@pytest.mark.parametrize("attention", ["shared", "sparse", "attend"])
def test_a_chain_of_launches_reads_what_was_just_written(attention):
    """Steps into the same buffers without a pause, each kernel launched while the one before still runs: every q,
    key and index entry that a step reads is the one just written."""
    P, n, hq, hkv, d, steps = 16, 64, 8, 2, 64, 48
    g = torch.Generator(device=DEV).manual_seed(8)
    lead = list(range(8))
    tables = [lead + [8 + 4 * i + j for j in range(4)] for i in range(n)]
    qkv = torch.randn(steps, n, (hq + 2 * hkv) * d, generator=g, device=DEV).half()
    ang = torch.rand(256, d // 2, generator=g, device=DEV) * 6
    rope = (torch.cos(ang), torch.sin(ang))
    kv = [len(lead) * P + 1] * n

    def run(pause):
        bk = B200PagedBackend(1, 8 + 4 * n, P, hkv, hq, d, device=DEV, validate="device")
        bk.k_pool[0].copy_(torch.randn(bk.k_pool[0].shape, generator=g.manual_seed(9), device=DEV))
        bk.v_pool[0].copy_(torch.randn(bk.v_pool[0].shape, generator=g, device=DEV))
        index = PageIndex(bk)
        index.rebuild(range(bk.num_blocks))
        q_out = torch.empty(n, hq, d, dtype=torch.float16, device=DEV)
        outs = torch.empty(steps, n, hq, d, dtype=torch.float16, device=DEV)
        metas = [build_meta(tables, [x + t for x in kv], [1] * n, P, device=DEV) for t in range(steps)]
        plan = {"shared": lambda m: bk.plan_shared(m, SharedPrefix([n], [8])),
                "sparse": lambda m: bk.plan_sparse(m, index, 5), "attend": lambda m: m}[attention]
        plans = [plan(m) for m in metas]
        slices = [[x.unflatten(1, (-1, d)) for x in s.split([hq * d, hkv * d, hkv * d], 1)] for s in qkv]
        torch.cuda.synchronize()
        for t in range(steps):
            if attention == "attend":
                bk.plan(metas[t])
            bk.rope_append(0, *slices[t], metas[t], rope, index=index, q_out=q_out)
            if pause:
                torch.cuda.synchronize()
            if attention == "shared":
                bk.attend_shared(q_out, 0, 0.125, plans[t], out=outs[t])
            elif attention == "sparse":
                bk.attend_sparse(q_out, 0, 0.125, plans[t], out=outs[t])
            else:
                bk.attend(q_out, 0, 0.125, metas[t], out=outs[t])
            if pause:
                torch.cuda.synchronize()
        bk.check_status()
        return outs

    want = run(True)
    for _ in range(3):
        assert torch.equal(run(False), want)


# ---------------------------------------------------------------- rope_append
def test_q_out_over_k_or_v_is_refused():
    """k or v may be read after a row of q_out has been written."""
    bk = B200PagedBackend(1, 8, 16, 2, 2, 64, device=DEV)
    meta = build_meta([[0, 1]], [20], [20], 16, device=DEV)
    rope = (torch.ones(32, 32, device=DEV), torch.zeros(32, 32, device=DEV))
    q, k, v = (torch.randn(20, 2, 64, device=DEV).half() for _ in range(3))
    for kw in (dict(k=k, v=v, q_out=k), dict(k=k, v=v, q_out=v)):
        with pytest.raises(ValueError, match="overlaps"):
            bk.rope_append(0, q, kw["k"], kw["v"], meta, rope, q_out=kw["q_out"])
    flat = torch.zeros(2 * q.numel() - 64, dtype=torch.float16, device=DEV)
    with pytest.raises(ValueError, match="overlaps"):  # k's last head is q_out's first
        bk.rope_append(0, q, flat[:q.numel()].view(q.shape), v, meta, rope, q_out=flat[-q.numel():].view(q.shape))
    qkv = torch.cat([q.flatten(1), k.flatten(1), v.flatten(1)], 1)
    qs, ks, vs = (x.unflatten(1, (-1, 64)) for x in qkv.split([128, 128, 128], 1))
    fits = torch.zeros(3 * q.numel(), dtype=torch.float16, device=DEV)  # neighbours that do not meet
    for args, out in (((qs, ks, vs), fits[:q.numel()].view(q.shape)), ((q, k, v), q)):
        got = bk.rope_append(0, *args, meta, rope, q_out=out)
        assert got is out
        slots = meta.slot_mapping.long()
        assert torch.equal(bk.k_pool[0].flatten(0, 1)[slots], k) and torch.equal(bk.v_pool[0].flatten(0, 1)[slots], v)


# ---------------------------------------------------------------- shared-prefix attention
@pytest.mark.parametrize("hq,hkv", [(32, 8), (4, 4)])
def test_rows_of_inconsistent_tables_are_zeros(hq, hkv):
    """Every row of out is written: zeros where the sequence's tables are refused, the others' results as ever."""
    fam = [(4, [(20, 1), (9, 3)]), (0, [(40, 5), (8, 1)]), (0, [(30, 2)]), (3, [(7, 1), (1, 1)])]
    bk, meta, q, shared, tables = sh.build(fam, hq, hkv, validate="device")
    want = sh.attend64(bk, meta, q, tables, 0.125)
    row_of = meta.batch_indices
    for bad in ([0], [1], [2, 3], [4], [5, 6], list(range(7))):
        kl = meta.kv_lens.clone()
        kl[bad] += 16
        out = torch.full_like(q, float("nan"))
        bk.attend_shared(q, 0, 0.125, bk.plan_shared(dataclasses.replace(meta, kv_lens=kl), shared), out=out)
        with pytest.raises(PkvError, match="inconsistent"):
            bk.check_status()
        refused = torch.isin(row_of, torch.tensor(bad, dtype=row_of.dtype, device=DEV))
        assert not out[refused].any()
        sh.close(out, torch.where(refused[:, None, None], 0.0, want), bk)
    # the step's own sums disagree: nothing is computed
    out = torch.full_like(q, float("nan"))
    bk.attend_shared(q, 0, 0.125, bk.plan_shared(dataclasses.replace(meta, cu_query_lens=meta.cu_query_lens + 1), shared),
                     out=out)
    with pytest.raises(PkvError, match="inconsistent"):
        bk.check_status()
    assert not out.any()


@pytest.mark.parametrize("where", [DEV, "cpu"])
@pytest.mark.parametrize("validate", ["host", "device"])
def test_plans_without_the_kernel_hold_their_tables(validate, where):
    """head_dim 32: a plan keeps its step when ``meta`` is overwritten in place, and the next plan sees the new one."""
    bk, meta, q, shared, tables = sh.build([(0, [(100, 1), (70, 5), (33, 1)])], 6, 2, validate=validate, d=32)
    meta = build_meta(tables, [100, 70, 33], [1, 5, 1], 16, device=where)
    first = bk.plan_shared(meta, shared)
    want = sh.attend64(bk, meta, q, tables, 0.2)
    sh.close(bk.attend_shared(q, 0, 0.2, first), want, bk)
    assert first.workspace is None
    other = [tables[0], tables[1], tables[0][:3]]  # the third sequence takes over pages of the first
    changed = build_meta(other, [99, 70, 48], [1, 5, 1], 16, device=where)
    for f in ("kv_lens", "positions", "kv_indptr", "kv_indices", "kv_last_page_len"):
        getattr(meta, f).copy_(getattr(changed, f))
    second = bk.plan_shared(meta, shared)
    sh.close(bk.attend_shared(q, 0, 0.2, second), sh.attend64(bk, meta, q, other, 0.2), bk)
    sh.close(bk.attend_shared(q, 0, 0.2, first), want, bk)
    bk.check_status()


@pytest.mark.parametrize("d,hq,hkv", [(32, 6, 2), (64, 6, 2), (128, 4, 4)])
@pytest.mark.parametrize("claim", ["other pages", "past the new tokens", "more pages than there are"])
def test_wrong_claims_without_the_kernel(claim, d, hq, hkv):
    fam = [(4, [(20, 1), (9, 1)]), (3, [(40, 5), (8, 1)])]
    pages = {"other pages": [5, 3], "past the new tokens": [4, 5], "more pages than there are": [4, 50]}[claim]
    bk, meta, q, shared, tables = sh.build(fam, hq, hkv, validate="device", d=d)
    out = bk.attend_shared(q, 0, 0.2, bk.plan_shared(meta, SharedPrefix([2, 2], pages)))
    with pytest.raises(PkvError, match="inconsistent"):
        bk.check_status()
    sh.close(out, sh.attend64(bk, meta, q, tables, 0.2), bk)
    bk.plan_shared(meta, shared)
    bk.check_status()


@pytest.mark.parametrize("pages", [0, 2])
def test_queries_that_are_not_numbers_give_no_numbers(pages):
    """A NaN in one query row reaches that row of out, and no other, shared or not."""
    bk, meta, q, shared, tables = sh.build([(pages, [(40, 5), (30, 1), (9, 2)])], 8, 2)
    q[1, 3, 7] = q[5, 0, 0] = q[6, 7, 63] = float("nan")
    out = bk.attend_shared(q, 0, 0.125, bk.plan_shared(meta, shared))
    bad = torch.zeros(q.shape[:2], dtype=torch.bool, device=DEV)
    bad[1, 3] = bad[5, 0] = bad[6, 7] = True
    assert bool(torch.isnan(out[bad]).all())
    want = sh.attend64(bk, meta, torch.where(bad[..., None], 0, q), tables, 0.125)
    sh.close(torch.where(bad[..., None], want.to(q.dtype), out), want, bk)


# ---------------------------------------------------------------- page index
GEOMETRIES = [(torch.float16, 16, 64), (torch.bfloat16, 16, 64), (torch.float32, 16, 64), (torch.float16, 16, 128),
              (torch.bfloat16, 32, 256), (torch.float32, 16, 128), (torch.float16, 5, 40), (torch.float32, 3, 33)]


@pytest.mark.parametrize("dtype,page,d", GEOMETRIES)
def test_index_of_keys_that_are_not_finite(dtype, page, d):
    """An infinite key: an infinite scale, 127 with its sign where a bound is infinite, 0 elsewhere. A key that is
    no number: neither is the scale, codes 0."""
    bk = B200PagedBackend(1, 9, page, 2, 2, d, device=DEV, dtype=dtype)
    k = bk.k_pool[0]
    k.copy_(torch.randn(k.shape, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV))
    inf, nan = float("inf"), float("nan")
    k[1, 2, 0, 5] = inf
    k[2, 0, 1, d - 1] = -inf
    k[3, :, 0, 7], k[3, page - 1, 0, 0] = inf, -inf
    k[4, :, 1, 9] = -inf
    k[5, 1, 0, 3] = nan
    k[6, page - 1, 1, d - 1], k[6, 0, 1, 0] = nan, inf
    k[7, :, :, :] = nan
    index = PageIndex(bk)
    index.rebuild(range(9))
    x = k.float().cpu().numpy()
    lo, hi = x.min(1), x.max(1)  # a NaN is the minimum and the maximum
    with np.errstate(invalid="ignore", divide="ignore"):
        scale = np.maximum(abs(lo), abs(hi)).max(-1) * np.float32(1 / 127)
        def code(b, up):
            y = np.clip((np.ceil if up else np.floor)(b / scale[..., None]), -127, 127)
            y = np.where(np.isinf(b), np.copysign(127, b), np.where(np.isinf(scale)[..., None], 0, y))
            return np.where(scale[..., None] > 0, y, 0)
        want = np.stack([code(lo, False), code(hi, True)], -2).astype(np.int8)
    assert np.array_equal(index.scales[0].cpu().numpy(), scale, equal_nan=True)
    assert np.array_equal(index.codes[0].cpu().numpy(), want)


@pytest.mark.parametrize("dtype,page,d", [(torch.float16, 16, 64), (torch.bfloat16, 16, 128), (torch.float32, 16, 64),
                                          (torch.float16, 8, 64)])
def test_pages_of_keys_that_are_not_finite(dtype, page, d):
    """Order of the scores: no number, then the infinite bound that the query reaches, then finite ones, then the
    bound of minus infinity; equal ones to the lower page."""
    bk, index, seqs, meta, q = sp.build([(page * 40, 1)], page, 2, 1, d, dtype)
    ids = seqs[0].block_ids
    q.copy_(torch.randn(q.shape, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).abs() + 0.1)
    k = bk.k_pool[0]
    k[ids[30], 1, 0, 4] = float("inf")   # positive query: +inf
    k[ids[10], 2, 0, 3] = float("inf")
    k[ids[20], 0, 0, 8] = float("nan")
    k[ids[25], 0, 0, 8] = float("-inf")  # 0 from that dim, 0 from the others: 0 * inf, no number
    k[ids[5], :, 0, 2] = float("-inf")   # whatever the key: -inf
    index.rebuild(ids)
    def chosen(budget):
        plan = bk.plan_sparse(meta, index, budget, sink=0, recent=1)
        return bk.select_pages(q, 0, plan)[0, 0].tolist()
    assert chosen(3) == [20, 25, 39]
    assert chosen(5) == [10, 20, 25, 30, 39]
    assert chosen(39) == [p for p in range(40) if p != 5]


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype,page,hq,d", [(torch.float16, 16, 8, 64), (torch.bfloat16, 16, 2, 128),
                                             (torch.float32, 16, 4, 64), (torch.float16, 16, 9, 64)])
def test_queries_that_are_not_finite_choose_the_lowest_pages(dtype, page, hq, d, value):
    """The scores of a KV head with such a query are no numbers: all equal. Other KV heads keep theirs."""
    bk, index, seqs, meta, q = sp.build([(page * 60, 1), (page * 50, 1)], page, 2 * hq, 2, d, dtype)
    plan = bk.plan_sparse(meta, index, 7, sink=1, recent=2)
    before = bk.select_pages(q, 0, plan)
    q[0, hq - 1, 5] = value
    after = bk.select_pages(q, 0, plan)
    assert after[0, 0].tolist() == [0, 1, 2, 3, 4, 58, 59]
    assert torch.equal(after[0, 1], before[0, 1]) and torch.equal(after[1], before[1])


class _Blocks:
    is_freed, seq_id = False, 0

    def __init__(self, ids, tokens):
        self.block_ids, self.num_tokens = ids, tokens


def _index_is_the_pools(bk, index, blocks):
    fresh = PageIndex(bk)
    fresh.rebuild(blocks)
    assert torch.equal(fresh.codes[:, blocks], index.codes[:, blocks])
    assert torch.equal(fresh.scales[:, blocks], index.scales[:, blocks])


@pytest.mark.parametrize("writer", ["append_kv", "append_attend decode", "append_attend prompt", "append_attend rope",
                                    "rope_append", "rope_append with another index", "copy_block", "copy_blocks",
                                    "swap_in", "reset"])
def test_every_writer_keeps_the_index(writer):
    """Blocks taken over from a former owner: their entries are the new keys', whoever wrote them."""
    from llm_serving_layer_b200 import B200SwapSpace
    P, hkv, hq, d, layers = 16, 2, 8, 64, 2
    bk = B200PagedBackend(layers, 12, P, hkv, hq, d, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(11)
    def fill():
        for pool in bk.k_pool + bk.v_pool:
            pool.copy_(torch.randn(pool.shape, generator=g, device=DEV))
    fill()
    index = PageIndex(bk)
    index.rebuild(range(12))
    old = index.codes.clone()
    tables, done = [[7, 2, 9], [4, 11]], [7, 2, 4, 11]
    def step(kv, new):
        m = build_meta(tables, kv, new, P, device=DEV)
        x = [torch.randn(sum(new), h, d, generator=g, device=DEV).half() for h in (hq, hkv, hkv)]
        return m, *x
    rope = (torch.randn(64, d // 2, device=DEV, generator=g), torch.randn(64, d // 2, device=DEV, generator=g))
    if writer.startswith("copy") or writer in ("swap_in", "reset"):
        if writer == "copy_block":
            for a, b in ((0, 7), (1, 2), (3, 4), (5, 11)):
                bk.copy_block(a, b)
        elif writer == "copy_blocks":
            bk.copy_blocks([0, 1, 3, 5], done)
        elif writer == "swap_in":
            space = B200SwapSpace(bk, synchronous=False)
            handle = space.swap_out("r", _Blocks([0, 1, 3, 5], 64))
            space.swap_in(handle, _Blocks(done, 64))
            space.wait()
        else:
            bk.reset()
            done = list(range(12))
    elif writer == "append_attend decode":
        m, q, k, v = step([35, 31], [35, 31])
        bk.append_kv(0, k, v, m)
        bk.append_kv(1, k, v, m)
        m, q, k, v = step([36, 32], [1, 1])
        for l in range(layers):
            bk.append_attend(l, k, v, q, 0.125, m)
    else:
        m, q, k, v = step([40, 32], [40, 32])
        other = PageIndex(bk) if writer == "rope_append with another index" else None
        for l in range(layers):
            if writer == "append_kv":
                bk.append_kv(l, k, v, m)
            elif writer == "append_attend prompt":
                bk.append_attend(l, k, v, q, 0.125, m)
            elif writer == "append_attend rope":
                bk.append_attend(l, k, v, q, 0.125, m, rope=rope)
            else:
                bk.rope_append(l, q, k, v, m, rope, index=other)
    bk.check_status()
    assert not torch.equal(index.codes[:, done], old[:, done])
    _index_is_the_pools(bk, index, done)


def test_an_index_that_is_gone_costs_nothing():
    bk = B200PagedBackend(1, 4, 16, 2, 2, 64, device=DEV)
    index = PageIndex(bk)
    assert len(bk._indexes) == 1
    del index
    assert not bk._indexes


# ---------------------------------------------------------------- pools beyond 4 GiB
def test_offsets_past_32_bits():
    """A K slab of more than 2^32 bytes: append, index and page-sparse attention at its end."""
    import test_gpu_rope_append as ra
    hkv, hq, d, P = 8, 8, 128, 16
    blocks = (1 << 32) // (P * hkv * d * 2) + 24
    bk = B200PagedBackend(1, blocks, P, hkv, hq, d, device=DEV, validate="device")
    ids = [blocks - 1 - i for i in range(20)]
    kv = P * 20 - 3
    meta = build_meta([ids], [kv], [kv], P, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    q, k, v = (torch.randn(kv, h, d, generator=g, device=DEV).half() for h in (hq, hkv, hkv))
    index, rope = PageIndex(bk), ra.tables(512, d)
    q = bk.rope_append(0, q, k, v, meta, rope, index=index)
    slots = meta.slot_mapping.long()
    kp, vp = bk.k_pool[0].flatten(0, 1), bk.v_pool[0].flatten(0, 1)
    ra.check_rotation(kp[slots], k, meta.positions, rope, False)
    assert torch.equal(vp[slots], v)
    assert not bk.k_pool[0][:1000].any() and not bk.v_pool[0][:1000].any()
    codes, scales = ra.entries(bk.k_pool[0][ids[:19]])
    assert np.array_equal(index.codes[0, ids[:19]].cpu().numpy(), codes)
    assert np.array_equal(index.scales[0, ids[:19]].cpu().numpy(), scales)

    class S:
        block_ids = ids
    last, step = q[-1:].contiguous(), build_meta([ids], [kv], [1], P, device=DEV)
    out, pages = bk.attend_sparse(last, 0, d ** -0.5, bk.plan_sparse(step, index, 6))
    bk.check_status()
    assert pages[0].tolist() == sp.choose(bk, index, [S], step, last, 6, 1, 1)[0]
    sp.close(out, sp.attend64(bk, [S], step, last, pages.tolist(), d ** -0.5), bk)


def test_shared_pages_past_32_bits():
    """... and shared pages, rests and chunks at its end."""
    hkv, hq, d, P = 8, 16, 64, 16
    blocks = (1 << 32) // (P * hkv * d * 2) + 40
    bk = B200PagedBackend(1, blocks, P, hkv, hq, d, device=DEV, validate="device")
    ids = [blocks - 1 - i for i in range(30)]
    tables = [ids[:9] + ids[9:12], ids[:9] + ids[12:20], ids[20:28]]
    kv, ql = [9 * P + 40, 9 * P + 120, 100], [1, 7, 1]
    g = torch.Generator(device=DEV).manual_seed(1)
    for pool in (bk.k_pool[0], bk.v_pool[0]):
        pool[ids] = torch.randn(30, P, hkv, d, generator=g, device=DEV).half()
    meta = build_meta(tables, kv, ql, P, device=DEV)
    q = torch.randn(9, hq, d, generator=g, device=DEV).half()
    out = bk.attend_shared(q, 0, 0.125, bk.plan_shared(meta, SharedPrefix([2, 1], [9, 0])))
    bk.check_status()
    want = sh.attend64(bk, meta, q, tables, 0.125)
    top = float(bk.v_pool[0][ids].abs().max())
    assert float((out.double() - want).abs().max()) <= (2 * 2.0 ** -11 + 2.0 ** -18) * top


@pytest.mark.parametrize("new", [300, 700])
def test_prompt_chunks_over_listed_pages(new):
    """Page-sparse attention of hundreds of new tokens of one sequence beside a decode row."""
    bk, index, seqs, meta, q = sp.build([(900, new), (400, 1)], 16, 4, 2, 64)
    plan = bk.plan_sparse(meta, index, 9, sink=1, recent=3)
    out, pages = bk.attend_sparse(q, 0, 0.125, plan)
    bk.check_status()
    want = sp.choose(bk, index, seqs, meta, q, 9, 1, 3)
    assert np.array_equal(pages.cpu().numpy(), np.array([[r + [-1] * (9 - len(r)) for r in row] for row in want]))
    sp.close(out, sp.attend64(bk, seqs, meta, q, want, 0.125), bk)


@pytest.mark.parametrize("new", [40, 700])
def test_tensor_memory_through_a_chain_of_launches(new):
    """Prompt attention and shared-prefix attention one after the other behind a kernel of some milliseconds, none
    of them with a pause: each holds tensor memory of its own."""
    bk, meta, q, shared, tables = sh.build([(21, [(4 + i % 37, 1 + i % 3) for i in range(40)]), (0, [(new, new)] * 6)],
                                           validate="device")
    plan = bk.plan_shared(meta, shared)
    slow = B200PagedBackend(1, 1, 1024, 1, 1, 64, device=DEV, dtype=torch.float32, validate="device")
    one = build_meta([[0]], [1024], [1], 1024, device=DEV)
    splan = slow.plan_sparse(one, PageIndex(slow), 100, max_pages=1)
    x, pages = torch.ones(1, 1, 64, device=DEV), torch.zeros((1, 1, 100), dtype=torch.int32, device=DEV)
    bk.plan(meta)
    want_a, want_s = bk.attend(q, 0, 0.125, meta), bk.attend_shared(q, 0, 0.125, plan)
    outs = [torch.empty_like(q) for _ in range(6)]
    torch.cuda.synchronize()
    slow.attend_pages(x, 0, 0.1, splan, pages)
    for i in range(0, 6, 2):
        bk.attend(q, 0, 0.125, meta, out=outs[i])
        bk.attend_shared(q, 0, 0.125, plan, out=outs[i + 1])
    bk.check_status()
    assert all(torch.equal(o, want_a) for o in outs[0::2]) and all(torch.equal(o, want_s) for o in outs[1::2])


# ---------------------------------------------------------------- plans
def test_plans_of_another_backend_are_refused():
    """A plan's page ids were checked against its own backend's pool, which may be larger."""
    bk, meta, q, shared, _ = sh.build(sh.CASES["one family"], 8, 2)
    index = PageIndex(bk)
    plans = bk.plan_shared(meta, shared), bk.plan_sparse(meta, index, 4)
    other = B200PagedBackend(1, 2, 16, 2, 8, 64, device=DEV)
    pages = torch.zeros(4, 2, 4, dtype=torch.int32, device=DEV)
    for call in (lambda: other.attend_shared(q, 0, 0.125, plans[0]), lambda: other.attend_sparse(q, 0, 0.125, plans[1]),
                 lambda: other.select_pages(q, 0, plans[1]), lambda: other.attend_pages(q, 0, 0.125, plans[1], pages)):
        with pytest.raises(ValueError, match="another backend"):
            call()
    small, meta, q, shared, _ = sh.build([(0, [(100, 1), (70, 5)])], 6, 2, d=32)  # attend's geometry
    plan = small.plan_shared(meta, shared)
    with pytest.raises(ValueError, match="another backend"):
        other.attend_shared(q, 0, 0.125, plan)


def test_plans_of_device_built_steps():
    """Steps assembled on the device into buffers that are used again: a plan holds its own copies."""
    from llm_serving_layer_b200 import DeviceBlockTables
    bk, meta, q, shared, tables = sh.build([(4, [(20, 1), (9, 3)]), (0, [(40, 5)])], 8, 2)
    bt = DeviceBlockTables(8, 16, 16, num_blocks=bk.num_blocks, device=DEV, ring=1)
    for i, t in enumerate(tables):
        bt.bind(i, t)
    index = PageIndex(bk)
    index.rebuild(sorted({p for t in tables for p in t[:2]}))
    want = bk.attend_shared(q, 0, 0.125, bk.plan_shared(meta, shared))
    want_s = bk.attend_sparse(q, 0, 0.125, bk.plan_sparse(meta, index, 3))
    step = bt.build_batch_meta([0, 1, 2], [1, 3, 5], [84, 73, 40])
    plan, sparse = bk.plan_shared(step, shared), bk.plan_sparse(step, index, 3)
    bt.build_batch_meta([2, 0, 1], [1, 1, 1], [12, 30, 25])  # into the same buffers
    assert torch.equal(bk.attend_shared(q, 0, 0.125, plan), want)
    got = bk.attend_sparse(q, 0, 0.125, sparse)
    assert torch.equal(got[0], want_s[0]) and torch.equal(got[1], want_s[1])
    bk.check_status()
    bt.check_status()


def test_workspaces_that_are_not_taken_over():
    """Too small, of another type or without the memory its shape says: the plan makes its own."""
    bk, meta, q, shared, tables = sh.build(sh.CASES["one family"], 8, 2)
    first = bk.plan_shared(meta, shared)
    n = first.workspace.numel()
    for ws in (first.workspace[:n - 1], torch.empty(n // 4, dtype=torch.float32, device=DEV),
               torch.empty(1, dtype=torch.uint8, device=DEV).expand(n), torch.empty(n, dtype=torch.uint8)):
        plan = bk.plan_shared(meta, shared, workspace=ws)
        assert plan.workspace is not ws and plan.workspace.numel() == n
    sh.close(bk.attend_shared(q, 0, 0.125, plan), sh.attend64(bk, meta, q, tables, 0.125), bk)
    assert bk.plan_shared(meta, shared, workspace=first.workspace).workspace is first.workspace

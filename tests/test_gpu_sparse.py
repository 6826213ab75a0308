"""
Page-sparse attention: the chosen pages must equal a brute-force selection
(whole-number scores, ties to the lower page), the output the 64-bit attention
over them.

Output bound: the kernel rounds each probability to the pool dtype (relative u:
2^-11 fp16, 2^-8 bf16; none for fp32 pools) and the result once more; with
weights that sum to 1 both errors are at most u * max|v|, and the fp32
accumulation adds a part in 2^-20 of max|v|: |err| <= (2 u + 2^-18) max|v|.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import FifoAllocator, Seq, meta_for
from llm_serving_layer_b200 import B200PagedBackend, PageIndex
from llm_serving_layer_b200._native import PkvError

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 0.0}


@pytest.fixture(scope="module", autouse=True)
def cuda():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device (run with -m 'not gpu' on CPU)"


def build(specs, page=16, hq=32, hkv=8, d=64, dtype=torch.float16, seed=0, poison=True, validate="host"):
    """(tokens held after the step, new tokens) per sequence. Unwritten tails
    and spare blocks hold NaN."""
    rs = np.random.RandomState(seed)
    blocks = sum(-(-kv // page) for kv, _ in specs) + 3
    alloc = FifoAllocator(blocks, page, order=rs.permutation(blocks))
    bk = B200PagedBackend(1, blocks, page, hkv, hq, d, device=DEV, dtype=dtype, validate=validate)
    g = torch.Generator(device=DEV).manual_seed(seed)
    base = torch.randn(blocks, 1, hkv, d, generator=g, device=DEV)
    bk.k_pool[0].copy_(base * 0.7 + 0.7 * torch.randn(blocks, page, hkv, d, generator=g, device=DEV))
    bk.v_pool[0].copy_(torch.randn(blocks, page, hkv, d, generator=g, device=DEV))
    seqs = []
    for i, (kv, _) in enumerate(specs):
        s = Seq(alloc, i)
        s.append(kv)
        seqs.append(s)
    index = PageIndex(bk)
    index.rebuild(range(blocks))
    if poison:
        written = torch.zeros(blocks * page, dtype=torch.bool, device=DEV)
        for s in seqs:
            written[[s.slot_for(p) for p in range(s.num_tokens)]] = True
        bk.k_pool[0].flatten(0, 1)[~written] = float("nan")
        bk.v_pool[0].flatten(0, 1)[~written] = float("nan")
    meta = meta_for(seqs, [q for _, q in specs], device=DEV)
    T = sum(q for _, q in specs)
    q = torch.randn(T, hq, d, generator=g, device=DEV).to(dtype)
    return bk, index, seqs, meta, q


def choose(bk, index, seqs, meta, q, budget, sink, recent):
    """Brute-force selection: lists of pages per token and KV head."""
    hkv, c = bk.n_kv_heads, np.float32(1.0 / 127.0)
    codes, scales = index.codes[0].cpu().numpy().astype(np.int64), index.scales[0].cpu().numpy()
    x = q.float().cpu().numpy().reshape(q.shape[0], hkv, -1, bk.head_dim)
    rows = []
    for s, t, pos in zip(meta.batch_indices.tolist(), range(q.shape[0]), meta.positions.tolist()):
        mine = pos // bk.block_size
        ids = np.asarray(seqs[s].block_ids[:mine + 1])
        row = []
        for h in range(hkv):
            qs = abs(x[t, h]).max(-1) * c
            q8 = np.clip(np.rint(x[t, h] / np.where(qs > 0, qs, 1)[:, None]), -127, 127).astype(np.int64)
            q8[qs == 0] = 0
            dot = np.maximum(q8[:, None] * codes[ids, h, 0], q8[:, None] * codes[ids, h, 1]).sum(-1)
            score = (dot.astype(np.float32) * qs[:, None]).max(0) * scales[ids, h]
            key = [(-np.inf if p < sink or p > mine - recent else -score[p], p) for p in range(mine + 1)]
            row.append(sorted(p for _, p in sorted(key)[:budget]))
        rows.append(row)
    return rows


def attend64(bk, seqs, meta, q, pages, scale):
    """64-bit attention over listed pages; zeros where nothing is visible."""
    P, hkv = bk.block_size, bk.n_kv_heads
    kp, vp = bk.k_pool[0].flatten(0, 1), bk.v_pool[0].flatten(0, 1)
    out = torch.zeros(q.shape[0], hkv, bk.n_heads // hkv, bk.head_dim, dtype=torch.float64, device=DEV)
    for t, (s, pos) in enumerate(zip(meta.batch_indices.tolist(), meta.positions.tolist())):
        for h in range(hkv):
            at = [seqs[s].block_ids[p] * P + o for p in pages[t][h] for o in range(P) if 0 <= p and p * P + o <= pos]
            if at:
                at = torch.tensor(at, device=DEV)
                w = torch.softmax(q[t].double().view(hkv, -1, bk.head_dim)[h] @ kp[at, h].double().T * scale, -1)
                out[t, h] = w @ vp[at, h].double()
    return out.view(q.shape)


def close(got, want, bk):
    top = float(torch.nan_to_num(bk.v_pool[0].float()).abs().max())
    bound = (2 * UNIT[bk.dtype] + 2.0 ** -18) * top
    err = float((got.double() - want).abs().max())
    assert err <= bound, (err, bound)


CASES = [
    # (kv, new) per sequence, budget, sink, recent
    ([(1, 1)], 4, 1, 1),
    ([(15, 1), (16, 1), (17, 1), (32, 1), (33, 1)], 2, 1, 1),
    ([(700, 1), (64, 1), (65, 1), (300, 1)], 8, 1, 2),
    ([(700, 1), (3, 1)], 64, 0, 1),                  # budget above the pages there are
    ([(1000, 7), (33, 33), (129, 5)], 6, 2, 3),      # several new tokens
    ([(5000, 1)], 37, 1, 1),                         # more pages than threads
    ([(2500, 3), (4097, 2)], 1, 0, 1),               # only the query's own page
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 64), (8, 8, 64), (6, 2, 128), (8, 1, 128), (5, 1, 64)])
@pytest.mark.parametrize("case", CASES)
def test_tensor_core_kernel(case, hq, hkv, d, dtype):
    specs, budget, sink, recent = case
    bk, index, seqs, meta, q = build(specs, 16, hq, hkv, d, dtype)
    plan = bk.plan_sparse(meta, index, budget, sink=sink, recent=recent)
    out, pages = bk.attend_sparse(q, 0, d ** -0.5, plan)
    bk.check_status()
    want = choose(bk, index, seqs, meta, q, budget, sink, recent)
    padded = np.array([[r + [-1] * (budget - len(r)) for r in row] for row in want])
    assert np.array_equal(pages.cpu().numpy(), padded)
    close(out, attend64(bk, seqs, meta, q, want, d ** -0.5), bk)
    # the two halves, on another stream, give the same bits
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = bk.select_pages(q, 0, plan)
        out2 = bk.attend_pages(q, 0, d ** -0.5, plan, again)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, pages) and torch.equal(out2, out)


@pytest.mark.parametrize("dtype,page,hq,hkv,d", [
    (torch.float32, 16, 8, 2, 64), (torch.float16, 16, 18, 2, 64), (torch.float16, 8, 8, 2, 64),
    (torch.bfloat16, 32, 8, 2, 64), (torch.float16, 48, 8, 4, 128), (torch.float16, 16, 4, 2, 96),
    (torch.float32, 5, 3, 1, 33), (torch.bfloat16, 16, 2, 2, 256)])
def test_other_geometries(dtype, page, hq, hkv, d):
    specs = [(700, 1), (page, 1), (page + 1, 2), (333, 4)]
    bk, index, seqs, meta, q = build(specs, page, hq, hkv, d, dtype)
    plan = bk.plan_sparse(meta, index, 7, sink=1, recent=2)
    out, pages = bk.attend_sparse(q, 0, d ** -0.5, plan)
    bk.check_status()
    want = choose(bk, index, seqs, meta, q, 7, 1, 2)
    assert np.array_equal(pages.cpu().numpy(), np.array([[r + [-1] * (7 - len(r)) for r in row] for row in want]))
    close(out, attend64(bk, seqs, meta, q, want, d ** -0.5), bk)


def test_ties_go_to_the_lower_page():
    bk, index, seqs, meta, q = build([(16 * 900, 1)], hq=4, hkv=1)
    index.codes.fill_(5)
    index.scales.fill_(0.5)
    pages = bk.select_pages(q, 0, bk.plan_sparse(meta, index, 300, sink=0, recent=1))
    assert pages[0, 0].tolist() == list(range(299)) + [899]
    index.codes[0, seqs[0].block_ids[700:720]] = 6  # 20 higher bounds (q has a positive sum or not: same for all)
    pages = bk.select_pages(q, 0, bk.plan_sparse(meta, index, 300, sink=2, recent=3))
    assert pages[0, 0].tolist() == choose(bk, index, seqs, meta, q, 300, 2, 3)[0][0]


def test_query_of_zeros_and_infinite_bounds():
    bk, index, seqs, meta, q = build([(16 * 40, 1)], hq=4, hkv=1)
    q.zero_()
    out, pages = bk.attend_sparse(q, 0, 0.125, bk.plan_sparse(meta, index, 8))
    assert pages[0, 0].tolist() == [0, 1, 2, 3, 4, 5, 6, 39]
    close(out, attend64(bk, seqs, meta, q, [[pages[0, 0].tolist()]], 0.125), bk)


def test_given_pages():
    """Rows that list nothing, list past the query, list a page twice, in any order."""
    bk, index, seqs, meta, q = build([(100, 3), (16, 1)], hq=8, hkv=2)
    plan = bk.plan_sparse(meta, index, 6)
    lists = [[[-1] * 6, [0, 6, 7, 900, -5, 3]], [[3, 1, 0, 5, 2, 4], [2, -1, -1, -1, -1, 0]],
             [[6, -1, -1, -1, -1, -1], [1, 1, -1, -1, -1, -1]], [[5, 4, 3, 2, 1, -1], [0, 1, -1, -1, -1, -1]]]
    pages = torch.tensor(lists, dtype=torch.int32, device=DEV)
    out = bk.attend_pages(q, 0, 0.125, plan, pages)
    bk.check_status()
    close(out, attend64(bk, seqs, meta, q, [[[p for p in r if 0 <= p < 7] for r in row] for row in lists], 0.125), bk)
    assert not out[0, :4].any()   # nothing listed
    assert not out[3, :4].any()   # only pages past the query's own
    keep = torch.full_like(q, 7.0)
    assert bk.attend_pages(q, 0, 0.125, plan, pages, out=keep) is keep and torch.equal(keep, out)


def test_negative_and_zero_scale():
    bk, index, seqs, meta, q = build([(200, 1)], hq=8, hkv=2)
    plan = bk.plan_sparse(meta, index, 5)
    for scale in (-0.125, 0.0):
        out, pages = bk.attend_sparse(q, 0, scale, plan)
        close(out, attend64(bk, seqs, meta, q, pages.tolist(), scale), bk)


def test_more_tokens_than_the_pool_dtype_counts():
    """A query's own page is the last of a long list: 64-bit offsets into a pool beyond 4 GiB."""
    hkv, d, blocks = 8, 128, 66000
    bk = B200PagedBackend(1, blocks, 16, hkv, 8, d, device=DEV, validate="device")
    ids = [blocks - 1 - i for i in range(20)]
    from llm_serving_layer_b200 import build_meta
    meta = build_meta([ids], [16 * 20 - 3], [1], 16, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    for pool in (bk.k_pool[0], bk.v_pool[0]):
        pool[ids] = torch.randn(20, 16, hkv, d, generator=g, device=DEV).half()
    index = PageIndex(bk)
    index.rebuild(ids)
    q = torch.randn(1, 8, d, generator=g, device=DEV).half()
    out, pages = bk.attend_sparse(q, 0, d ** -0.5, bk.plan_sparse(meta, index, 6))
    bk.check_status()

    class S:
        block_ids = ids
    assert pages[0].tolist() == choose(bk, index, [S], meta, q, 6, 1, 1)[0]
    close(out, attend64(bk, [S], meta, q, pages.tolist(), d ** -0.5), bk)


def test_inconsistent_tables_are_flagged():
    import dataclasses
    bk, index, seqs, meta, q = build([(100, 1), (50, 1)], hq=8, hkv=2, validate="device")
    bad = meta.kv_indices.clone()
    bad[1] = bk.num_blocks
    plan = bk.plan_sparse(dataclasses.replace(meta, kv_indices=bad), index, 3, max_pages=7)
    bk.attend_sparse(q, 0, 0.125, plan)
    with pytest.raises(PkvError, match="outside the pool"):
        bk.check_status()
    plan = bk.plan_sparse(dataclasses.replace(meta, kv_lens=meta.kv_lens + 1), index, 3, max_pages=7)
    out, pages = bk.attend_sparse(q, 0, 0.125, plan)
    assert not out.any() and bool((pages == -1).all())
    with pytest.raises(PkvError, match="inconsistent"):
        bk.check_status()
    plan = bk.plan_sparse(meta, index, 3, max_pages=4)  # a sequence longer than announced
    out, pages = bk.attend_sparse(q, 0, 0.125, plan)
    assert not out[0].any() and bool((pages[0] == -1).all()) and bool(out[1].any())
    with pytest.raises(PkvError, match="inconsistent"):
        bk.check_status()


def test_refusals():
    bk, index, seqs, meta, q = build([(100, 1)], hq=8, hkv=2)
    for kw in (dict(budget=0), dict(budget=2, sink=2), dict(budget=4, recent=0), dict(budget=4, sink=-1)):
        with pytest.raises(ValueError, match="budget"):
            bk.plan_sparse(meta, index, **kw)
    with pytest.raises(ValueError, match="max_pages"):
        bk.plan_sparse(meta, index, 4, max_pages=0)
    other = build([(100, 1)], hq=8, hkv=2)
    with pytest.raises(ValueError, match="another backend"):
        bk.plan_sparse(meta, other[1], 4)
    plan = bk.plan_sparse(meta, index, 4)
    with pytest.raises(ValueError, match="q has shape"):
        bk.attend_sparse(q[:, :4], 0, 0.125, plan)
    with pytest.raises(ValueError, match="layer_idx"):
        bk.attend_sparse(q, 1, 0.125, plan)
    with pytest.raises(ValueError, match="pages must be"):
        bk.attend_pages(q, 0, 0.125, plan, torch.zeros(1, 2, 5, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="out must be"):
        bk.attend_sparse(q, 0, 0.125, plan, out=q.float())
    with pytest.raises(PkvError, match="shared memory"):
        bk.attend_sparse(q, 0, 0.125, bk.plan_sparse(meta, index, 4, max_pages=1 << 20))

"""
Shared-prefix attention against the 64-bit attention over each sequence's own
page list: the result must not depend on what is shared.

Bound: as the other attention kernels, each probability is rounded to the pool
dtype (relative u: 2^-11 fp16, 2^-8 bf16) and the result once more, both at most
u * max|v| with weights that sum to 1; the fp32 pieces and their merge add a part
in 2^-18: |err| <= (2 u + 2^-18) max|v|.
"""

from __future__ import annotations

import dataclasses

import numpy as np
import pytest
import torch

from llm_serving_layer_b200 import B200PagedBackend, SharedPrefix, build_meta
from llm_serving_layer_b200._native import PkvError

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module", autouse=True)
def cuda():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device (run with -m 'not gpu' on CPU)"


def build(families, hq=32, hkv=8, dtype=torch.float16, seed=0, validate="host", layers=1, d=64):
    """``families``: (shared pages, [(tokens after the shared pages, new tokens)]).
    Unwritten tails and spare blocks hold NaN."""
    rs = np.random.RandomState(seed)
    need = sum(p + sum(-(-t // 16) for t, _ in members) for p, members in families) + 3
    ids = rs.permutation(need).tolist()
    at, tables, kv, ql, written = 0, [], [], [], []
    for p, members in families:
        lead, at = ids[at:at + p], at + p
        for tail, new in members:
            n = -(-tail // 16)
            tables.append(lead + ids[at:at + n])
            at += n
            kv.append(p * 16 + tail)
            ql.append(new)
            written += [tables[-1][i // 16] * 16 + i % 16 for i in range(kv[-1])]
    bk = B200PagedBackend(layers, need, 16, hkv, hq, d, device=DEV, dtype=dtype, validate=validate)
    g = torch.Generator(device=DEV).manual_seed(seed)
    live = torch.zeros(need * 16, dtype=torch.bool, device=DEV)
    live[written] = True
    for l in range(layers):
        for pool in (bk.k_pool[l], bk.v_pool[l]):
            pool.copy_(torch.randn(need, 16, hkv, d, generator=g, device=DEV))
            pool.flatten(0, 1)[~live] = float("nan")
    meta = build_meta(tables, kv, ql, 16, device=DEV)
    q = torch.randn(sum(ql), hq, d, generator=g, device=DEV).to(dtype)
    shared = SharedPrefix([len(m) for _, m in families], [p for p, _ in families])
    return bk, meta, q, shared, tables


def attend64(bk, meta, q, tables, scale, layer=0):
    hkv = bk.n_kv_heads
    kp, vp = bk.k_pool[layer].flatten(0, 1), bk.v_pool[layer].flatten(0, 1)
    out = torch.empty(q.shape, dtype=torch.float64, device=DEV)
    for t, (s, pos) in enumerate(zip(meta.batch_indices.tolist(), meta.positions.tolist())):
        at = torch.arange(pos + 1)
        at = (torch.tensor(tables[s])[at // 16] * 16 + at % 16).to(DEV)
        x = q[t].double().view(hkv, -1, bk.head_dim)
        w = torch.softmax(torch.einsum("hgd,khd->hgk", x, kp[at].double()) * scale, -1)
        out[t] = torch.einsum("hgk,khd->hgd", w, vp[at].double()).reshape(bk.n_heads, bk.head_dim)
    return out


def close(got, want, bk, layer=0):
    top = float(torch.nan_to_num(bk.v_pool[layer].float()).abs().max())
    err, bound = float((got.double() - want).abs().max()), (2 * UNIT[bk.dtype] + 2.0 ** -18) * top
    assert err <= bound, (err, bound)


CASES = {
    "two rows, one page": [(1, [(1, 1), (16, 1)])],
    "one family": [(64, [(5, 1), (40, 1), (16, 1), (17, 1)])],
    "families and loners": [(3, [(1, 1)] * 3), (0, [(70, 1)]), (17, [(33, 1)] * 5), (9, [(20, 1)]), (0, [(3, 1), (4, 1)])],
    "more rows than a tile": [(21, [(1 + i % 37, 1) for i in range(150)])],
    "long prefix, ranges": [(700, [(9, 1), (200, 1), (31, 1)])],
    "several new tokens": [(20, [(5, 5), (64, 9), (70, 3)]), (6, [(40, 33), (2, 2)])],
    "chunks and decode rows": [(20, [(5, 1), (64, 40), (70, 1), (7, 7)]), (0, [(100, 50)]), (33, [(1, 1)] * 2)],
    "long own parts": [(8, [(3000, 1), (1500, 4), (2, 1)])],
    "no sharing": [(0, [(100, 1), (30, 20), (1, 1)])],
}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv", [(32, 8), (8, 8), (8, 4), (8, 1), (3, 3)])
@pytest.mark.parametrize("case", list(CASES))
def test_matches_unshared_attention(case, hq, hkv, dtype):
    bk, meta, q, shared, tables = build(CASES[case], hq, hkv, dtype)
    plan = bk.plan_shared(meta, shared)
    out = bk.attend_shared(q, 0, 0.125, plan)
    bk.check_status()
    close(out, attend64(bk, meta, q, tables, 0.125), bk)
    again = bk.attend_shared(q, 0, 0.125, plan)  # the plan's counters are left as they were; same bits
    assert torch.equal(again, out)


def test_more_rows_than_the_workspace_holds_pieces_for():
    """17000 sequences over one shared page: computed without sharing, same result."""
    n = 17000
    bk = B200PagedBackend(1, n + 1, 16, 1, 1, 64, device=DEV, validate="device")
    g = torch.Generator(device=DEV).manual_seed(5)
    for pool in (bk.k_pool[0], bk.v_pool[0]):
        pool.copy_(torch.randn(pool.shape, generator=g, device=DEV))
    tails = [1 + i % 16 for i in range(n)]
    meta = build_meta([[0, i + 1] for i in range(n)], [16 + t for t in tails], [1] * n, 16, device=DEV)
    q = torch.randn(n, 1, 64, generator=g, device=DEV).half()
    out = bk.attend_shared(q, 0, 0.125, bk.plan_shared(meta, SharedPrefix([n], [1])))
    bk.check_status()
    k = torch.cat([bk.k_pool[0][0, :, 0].expand(n, 16, 64), bk.k_pool[0][1:, :, 0]], 1).double()
    v = torch.cat([bk.v_pool[0][0, :, 0].expand(n, 16, 64), bk.v_pool[0][1:, :, 0]], 1).double()
    w = torch.einsum("nd,nkd->nk", q[:, 0].double(), k) * 0.125
    w = w.masked_fill(torch.arange(32, device=DEV) >= 16 + torch.tensor(tails, device=DEV)[:, None], -float("inf"))
    close(out[:, 0], torch.einsum("nk,nkd->nd", torch.softmax(w, -1), v), bk)


def test_many_sequences_in_families():
    """More sequences and families than the plan has threads, mixed with chunks."""
    fam = [(1 + i % 3, [(1 + (7 * i + j) % 40, 1) for j in range(1 + i % 4)]) for i in range(1100)]
    fam[5] = (2, [(30, 30), (9, 1)])
    bk, meta, q, shared, tables = build(fam, hq=4, hkv=2, validate="device")
    out = bk.attend_shared(q, 0, 0.125, bk.plan_shared(meta, shared))
    bk.check_status()
    want = bk.attend(q, 0, 0.125, meta)  # the plain path, itself held to the oracle elsewhere
    top = float(torch.nan_to_num(bk.v_pool[0].float()).abs().max())
    assert float((out.double() - want.double()).abs().max()) <= (4 * UNIT[bk.dtype] + 2.0 ** -17) * top


def test_layers_workspaces_and_streams():
    fam = CASES["chunks and decode rows"]
    bk, meta, q, shared, tables = build(fam, layers=3, validate="device")
    plan = bk.plan_shared(meta, shared)
    outs = [bk.attend_shared(q, l, 0.125, plan) for l in range(3)]
    for l in range(3):
        close(outs[l], attend64(bk, meta, q, tables, 0.125, l), bk, l)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        keep = torch.full_like(q, 9.0)
        second = bk.plan_shared(meta, shared, workspace=plan.workspace)
        assert second.workspace is plan.workspace
        assert bk.attend_shared(q, 1, 0.125, second, out=keep) is keep
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(keep, outs[1])
    bk.check_status()


def test_large_scores_and_scales():
    """Score ranges that rescale the running maximum, a zero and a negative scale."""
    bk, meta, q, shared, tables = build(CASES["long prefix, ranges"])
    bk.k_pool[0].mul_(8.0)
    plan = bk.plan_shared(meta, shared)
    for scale in (0.5, 0.0, -0.125):
        close(bk.attend_shared(q, 0, scale, plan), attend64(bk, meta, q, tables, scale), bk)


def test_geometries_without_the_kernel_run_attend():
    bk, meta, q, shared, tables = build(CASES["several new tokens"], hq=6, hkv=2, d=32)
    plan = bk.plan_shared(meta, shared)
    close(bk.attend_shared(q, 0, 0.2, plan), attend64(bk, meta, q, tables, 0.2), bk)
    assert bk.last_kernel == "generic"


@pytest.mark.parametrize("claim", ["other pages", "past the new tokens", "more pages than there are"])
def test_wrong_claims(claim):
    """Refused on the host; on the device computed without sharing, and flagged."""
    fam = [(4, [(20, 1), (9, 1)]), (3, [(40, 5), (8, 1)])]
    pages = {"other pages": [5, 3], "past the new tokens": [4, 5], "more pages than there are": [4, 50]}[claim]
    for validate in ("host", "device"):
        bk, meta, q, shared, tables = build(fam, validate=validate)
        wrong = SharedPrefix([2, 2], pages)
        if validate == "host":
            with pytest.raises(ValueError, match="group"):
                bk.plan_shared(meta, wrong)
            continue
        out = bk.attend_shared(q, 0, 0.125, bk.plan_shared(meta, wrong))
        with pytest.raises(PkvError):
            bk.check_status()
        close(out, attend64(bk, meta, q, tables, 0.125), bk)


def test_inconsistent_tables_are_flagged():
    bk, meta, q, shared, tables = build(CASES["one family"], validate="device")
    for change in (dict(kv_lens=meta.kv_lens + 16), dict(kv_last_page_len=torch.zeros_like(meta.kv_last_page_len)),
                   dict(kv_indices=torch.full_like(meta.kv_indices, bk.num_blocks))):
        bk.attend_shared(q, 0, 0.125, bk.plan_shared(dataclasses.replace(meta, **change), shared))
        with pytest.raises(PkvError):
            bk.check_status()


def test_refusals():
    bk, meta, q, shared, tables = build(CASES["one family"])
    with pytest.raises(ValueError, match="groups hold 3"):
        bk.plan_shared(meta, SharedPrefix([3], [1]))
    plan = bk.plan_shared(meta, shared)
    with pytest.raises(ValueError, match="q has shape"):
        bk.attend_shared(q[:2], 0, 0.125, plan)
    with pytest.raises(ValueError, match="layer_idx"):
        bk.attend_shared(q, 1, 0.125, plan)
    with pytest.raises(ValueError, match="overlap"):
        bk.attend_shared(q, 0, 0.125, plan, out=q)

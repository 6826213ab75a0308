"""
Host-side checks of the paged-cache operators without a GPU: families found from
block tables, and the refusals of the C entry points before any device call.
"""

from __future__ import annotations

import ctypes

import pytest

from llm_serving_layer_b200 import SharedPrefix
from llm_serving_layer_b200 import _native as N
from llm_serving_layer_b200 import build as B


@pytest.fixture(scope="module")
def lib():
    B.build()
    return N.lib()


def pool(dtype=0, n_kv=8, d=64, page=16, blocks=64, layers=2):
    return ctypes.byref(N.PoolDesc(0x1000, blocks, layers, page, n_kv, d, dtype, 0))


def index(codes=0x1000, scales=0x2000):
    return ctypes.byref(N.PageIndexDesc(codes, scales))


def test_families_from_block_tables():
    P = 16
    # a family of three over 2 pages, a loner, a pair whose second member holds only 1 whole page before its tokens
    tables = [[5, 6, 1], [5, 6, 2], [5, 6, 3], [9, 4], [7, 8, 10], [7, 8]]
    kv, ql = [40, 33, 40, 20, 40, 32], [1, 1, 8, 1, 1, 16]
    s = SharedPrefix.from_tables(tables, kv, ql, P)
    assert s.group_sizes == [3, 1, 2] and s.prefix_pages == [2, 0, 1]
    # joining must not cost more than it saves: 5 pages shared by two against 1 page shared by three
    s = SharedPrefix.from_tables([[1, 2, 3, 4, 5, 9], [1, 2, 3, 4, 5, 8], [1, 7, 6]], [96, 96, 48], [1, 1, 1], P)
    assert s.group_sizes == [2, 1] and s.prefix_pages == [5, 0]
    # ... but three over 3 pages beat two over 4
    s = SharedPrefix.from_tables([[1, 2, 3, 4, 9], [1, 2, 3, 4, 8], [1, 2, 3, 7]], [80, 80, 64], [1, 1, 1], P)
    assert s.group_sizes == [3] and s.prefix_pages == [3]
    # the query's own page is never shared, nor one a chunk is being written to
    s = SharedPrefix.from_tables([[1], [1]], [16, 16], [1, 1], P)
    assert s.group_sizes == [1, 1] and s.prefix_pages == [0, 0]
    assert SharedPrefix.from_tables([[3]], [1], [1], P).n_seqs == 1


def test_family_refusals():
    for bad in (([], []), ([1], []), ([0], [1]), ([2], [-1])):
        with pytest.raises(ValueError):
            SharedPrefix(*bad)
    with pytest.raises(ValueError):
        SharedPrefix.from_tables([[1]], [1, 2], [1], 16)


def test_rope_append_refusals(lib):
    def call(p=pool(), layer=0, q=0x1000, qs=2048, qo=0x1000, hq=32, k=0x1000, ks=512, v=0x1000, vs=512, slots=0x1000,
             pos=0x1000, n=4, cos=0x1000, sin=0x1000, rows=10, rot=64, ix=None):
        return lib.pkv_rope_append(p, layer, q, qs, qo, hq, k, ks, v, vs, slots, pos, n, cos, sin, rows, rot, 0, ix,
                                   None, None)

    for kw, rc in ((dict(p=None), N.PKV_ERR_ARG), (dict(layer=2), N.PKV_ERR_ARG), (dict(n=-1), N.PKV_ERR_ARG),
                   (dict(hq=-1), N.PKV_ERR_ARG), (dict(rot=63), N.PKV_ERR_ARG), (dict(rot=66), N.PKV_ERR_ARG),
                   (dict(rot=0), N.PKV_ERR_ARG), (dict(qs=2047), N.PKV_ERR_ARG), (dict(ks=511), N.PKV_ERR_ARG),
                   (dict(vs=0), N.PKV_ERR_ARG), (dict(q=None), N.PKV_ERR_ARG), (dict(slots=None), N.PKV_ERR_ARG),
                   (dict(cos=None), N.PKV_ERR_ARG), (dict(rows=0), N.PKV_ERR_ARG),
                   (dict(ix=index(None)), N.PKV_ERR_ARG), (dict(ix=index(0x1008)), N.PKV_ERR_ARG),
                   (dict(p=pool(dtype=3)), N.PKV_ERR_UNSUPPORTED)):
        assert call(**kw) == rc, kw
        assert lib.pkv_last_error()
    assert call(n=0) == N.PKV_OK  # nothing to append launches nothing


def test_index_refusals(lib):
    up, re = lib.pkv_page_index_update, lib.pkv_page_index_rebuild
    assert up(pool(), index(), 2, 0x1000, 4, None, None) == N.PKV_ERR_ARG
    assert up(pool(), index(), 0, None, 4, None, None) == N.PKV_ERR_ARG
    assert up(pool(), index(), 0, 0x1000, -1, None, None) == N.PKV_ERR_ARG
    assert up(pool(), None, 0, 0x1000, 4, None, None) == N.PKV_ERR_ARG
    assert up(pool(d=264), index(), 0, 0x1000, 4, None, None) == N.PKV_ERR_UNSUPPORTED
    assert up(pool(), index(), 0, None, 0, None, None) == N.PKV_OK
    assert re(pool(dtype=3), index(), 0x1000, 4, None, None) == N.PKV_ERR_UNSUPPORTED
    assert re(pool(), index(), None, 4, None, None) == N.PKV_ERR_ARG
    assert re(pool(), index(), None, 0, None, None) == N.PKV_OK


def batch(n=2, t=2, pages=4, cu=0x1000, ix=0x1000):
    return ctypes.byref(N.BatchDesc(n, t, pages, cu, 0x1000, 0x1000, ix, 0x1000, None))


def test_sparse_refusals(lib):
    def call(p=pool(), ix=index(), layer=0, hq=32, q=0x1000, out=0x1000, pages=0x1000, budget=8, sink=1, recent=1,
             b=batch(), rows=0x1000, most=4, mode=3):
        return lib.pkv_attend_sparse(p, ix, layer, hq, q, out, pages, 0.125, budget, sink, recent, b, rows, most, mode,
                                     None)

    for kw, rc in ((dict(layer=-1), 1), (dict(hq=30), 1), (dict(mode=0), 1), (dict(mode=4), 1), (dict(budget=0), 1),
                   (dict(sink=8), 1), (dict(recent=0), 1), (dict(ix=None), 1), (dict(b=None), 1),
                   (dict(b=batch(n=0)), 1), (dict(b=batch(t=-1)), 1),
                   (dict(b=batch(ix=None)), 1), (dict(q=None), 1), (dict(out=None), 1), (dict(pages=None), 1),
                   (dict(rows=None), 1), (dict(most=0), 1), (dict(p=pool(dtype=3)), 2), (dict(p=pool(d=512)), 2)):
        assert call(**kw) == rc, kw
    assert call(b=batch(t=0)) == N.PKV_OK

    def plan(p=pool(), b=batch(), bi=0x1000, most=4, rows=0x1000):
        return lib.pkv_plan_sparse(p, b, bi, most, rows, None)

    for kw in (dict(p=None), dict(b=None), dict(b=batch(n=0)), dict(b=batch(cu=None)), dict(bi=None), dict(most=0),
               dict(rows=None), dict(rows=0x1008)):
        assert plan(**kw) == N.PKV_ERR_ARG, kw
    assert plan(b=batch(t=0)) == N.PKV_OK


def test_shared_refusals(lib):
    size = lib.pkv_shared_workspace_size(pool(), 32, 2, 2, 4)
    assert size > 0 and lib.pkv_shared_workspace_size(None, 32, 2, 2, 4) == 0

    def plan(p=pool(), hq=32, b=batch(), groups=1, gi=0x1000, pp=0x1000, ws=0x1000, n=size):
        return lib.pkv_plan_shared(p, hq, b, groups, gi, pp, ws, n, None)

    for kw, rc in ((dict(hq=30), 1), (dict(b=None), 1), (dict(groups=0), 1), (dict(groups=3), 1), (dict(gi=None), 1),
                   (dict(pp=None), 1), (dict(ws=None), 1), (dict(n=size - 1), 1), (dict(ws=0x1010), 1),
                   (dict(b=batch(n=0)), 1), (dict(p=pool(d=128)), 2), (dict(p=pool(page=32)), 2),
                   (dict(p=pool(dtype=2)), 2), (dict(hq=24), 2)):
        assert plan(**kw) == rc, kw

    def attend(p=pool(), layer=0, q=0x1000, out=0x1000, b=batch(), ws=0x1000, n=size):
        return lib.pkv_attend_shared_planned(p, layer, 32, q, out, 0.125, b, ws, n, None)

    for kw, rc in ((dict(layer=2), 1), (dict(q=None), 1), (dict(q=0x1008), 1), (dict(out=None), 1), (dict(n=0), 1),
                   (dict(p=pool(d=128)), 2)):
        assert attend(**kw) == rc, kw
    assert attend(b=batch(t=0)) == N.PKV_OK


def test_shared_check_refusals(lib):
    def check(p=pool(d=128), b=batch(), groups=1, gi=0x1000, pp=0x1000):
        return lib.pkv_check_shared(p, b, groups, gi, pp, None)

    for kw in (dict(p=None), dict(b=None), dict(b=batch(n=0)), dict(b=batch(t=-1)), dict(b=batch(cu=None)),
               dict(b=batch(ix=None)), dict(groups=0), dict(groups=3), dict(gi=None), dict(pp=None)):
        assert check(**kw) == N.PKV_ERR_ARG, kw
    for p, hq in ((pool(d=128), 32), (pool(page=32), 32), (pool(dtype=2), 32), (pool(), 24), (pool(n_kv=9), 36)):
        assert lib.pkv_shared_workspace_size(p, hq, 2, 2, 4) == 0  # geometries that attend serves

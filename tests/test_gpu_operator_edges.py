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

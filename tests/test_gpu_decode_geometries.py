"""
Decode launches of pools with different KV head counts and the same query heads
per KV head, in turn: the kernel's shared-memory limit belongs to the function,
so preparing it for the smaller pool must not refuse the larger one's launches.
"""

from __future__ import annotations

import pytest
import torch

from llm_serving_layer_b200 import B200PagedBackend, build_meta

pytestmark = pytest.mark.gpu


def test_pools_of_different_kv_heads_in_turn():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device (run with -m 'not gpu' on CPU)"
    sides = []
    for hkv in (8, 2):
        bk = B200PagedBackend(1, 4, 16, hkv, hkv, 64, device="cuda:0")
        g = torch.Generator(device="cuda:0").manual_seed(hkv)
        bk.v_pool[0].copy_(torch.randn(bk.v_pool[0].shape, generator=g, device="cuda:0"))
        q = torch.zeros(1, hkv, 64, dtype=torch.float16, device="cuda:0")
        sides.append((bk, q))
    for bk, q in sides + sides:
        meta = build_meta([[2, 0]], [20], [1], 16, device="cuda:0")
        out = bk.attend(q, 0, 0.125, meta)  # zero queries: the mean of the 20 values
        assert bk.last_kernel == "decode"
        want = bk.v_pool[0][[2, 0]].flatten(0, 1)[:20].double().mean(0)
        assert float((out[0].double() - want).abs().max()) <= 2 * 2.0 ** -11 * 5

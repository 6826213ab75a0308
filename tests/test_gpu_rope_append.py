"""
``B200PagedBackend.rope_append`` and ``PageIndex``.

The rotation is held to the formula in 64 bits: the kernel computes
``a*c - b*s`` in fp32 (each product and the difference rounded, so an absolute
error of at most 3 * 2^-24 * (|a c| + |b s|)) and rounds once to the pool dtype
(relative 2^-11 for fp16, 2^-8 for bf16, 2^-24 for fp32). Where ``rope`` and
``append_kv`` exist for the same arguments the bits must be theirs. Index entries
are whole numbers computed from the keys the pool holds and must be equal.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import FifoAllocator, Seq, meta_for, slots_meta
from llm_serving_layer_b200 import B200PagedBackend, PageIndex
from llm_serving_layer_b200._native import PkvError

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROUND = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


@pytest.fixture(scope="module", autouse=True)
def cuda():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device (run with -m 'not gpu' on CPU)"


def tables(max_pos, dims, theta=10000.0):
    inv = theta ** (-torch.arange(0, dims, 2, dtype=torch.float32) / dims)
    ang = torch.arange(max_pos, dtype=torch.float32)[:, None] * inv
    return torch.cos(ang).to(DEV), torch.sin(ang).to(DEV)


def step(specs, page=16, hq=8, hkv=2, d=64, dtype=torch.float16, seed=0, layers=2, spare=4):
    """(tokens held, new tokens) per sequence over a scattered pool; q, k, v are
    slices of one fused tensor."""
    rs = np.random.RandomState(seed)
    blocks = sum(-(-(a + b) // page) for a, b in specs) + spare
    alloc = FifoAllocator(blocks, page, order=rs.permutation(blocks))
    seqs = []
    for i, (a, b) in enumerate(specs):
        s = Seq(alloc, i)
        s.append(a + b)
        seqs.append(s)
    bk = B200PagedBackend(layers, blocks, page, hkv, hq, d, device=DEV, dtype=dtype)
    g = torch.Generator(device=DEV).manual_seed(seed)
    for l in range(layers):
        bk.k_pool[l].copy_(torch.randn(blocks, page, hkv, d, generator=g, device=DEV))
        bk.v_pool[l].copy_(torch.randn(blocks, page, hkv, d, generator=g, device=DEV))
    meta = meta_for(seqs, [b for _, b in specs], device=DEV)
    T = sum(b for _, b in specs)
    fused = torch.randn(T, (hq + 2 * hkv) * d, generator=g, device=DEV).to(dtype)
    q, k, v = (x.unflatten(1, (-1, d)) for x in fused.split([hq * d, hkv * d, hkv * d], 1))
    return bk, meta, q, k, v


def rotated(x, pos, cos, sin, interleaved):
    """64-bit rotation and the sum of magnitudes its fp32 rounding scales with."""
    rot = 2 * cos.shape[1]
    c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
    y, mag = x.double().clone(), x.double().abs()
    ia = slice(0, rot, 2) if interleaved else slice(0, rot // 2)
    ib = slice(1, rot, 2) if interleaved else slice(rot // 2, rot)
    a, b = x[..., ia].double(), x[..., ib].double()
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    mag[..., ia], mag[..., ib] = (a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()
    return y, mag


def check_rotation(got, x, pos, rope, interleaved):
    want, mag = rotated(x, pos, *rope, interleaved)
    bound = ROUND[got.dtype] * want.abs() + 3 * 2.0 ** -24 * mag * (1 + ROUND[got.dtype]) + 2.0 ** -24
    assert bool(((got.double() - want).abs() <= bound).all())


CASES = [
    # specs, page, hq, hkv, d, rotary dims, interleaved
    ([(0, 1)], 16, 8, 2, 64, 64, False),
    ([(31, 1), (0, 1), (15, 1)], 16, 32, 8, 64, 64, False),
    ([(5, 45), (16, 1), (0, 33)], 16, 32, 8, 64, 64, False),
    ([(5, 45), (16, 1)], 16, 24, 8, 128, 96, True),
    ([(5, 45), (16, 1)], 16, 4, 1, 128, 128, True),
    ([(3, 30)], 16, 4, 4, 128, 64, False),
    ([(3, 30), (7, 2)], 8, 6, 2, 40, 40, False),     # rows of 80 bytes: vectors, half of 20 pairs not
    ([(3, 30), (7, 2)], 5, 3, 3, 34, 10, True),      # nothing aligned
    ([(3, 30), (7, 2)], 32, 2, 1, 256, 16, False),
    ([(0, 700), (1, 1300)], 16, 8, 2, 64, 64, False),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", CASES)
def test_rotation_and_append(case, dtype):
    specs, page, hq, hkv, d, rot, inter = case
    bk, meta, q, k, v = step(specs, page, hq, hkv, d, dtype)
    rope = tables(2048, rot)
    held = [p.clone() for p in bk.k_pool + bk.v_pool]
    got = bk.rope_append(1, q, k, v, meta, rope, interleaved=inter)
    bk.check_status()
    pos, slots = meta.positions, meta.slot_mapping.long()
    check_rotation(got, q, pos, rope, inter)
    kp, vp = bk.k_pool[1].flatten(0, 1), bk.v_pool[1].flatten(0, 1)
    check_rotation(kp[slots], k, pos, rope, inter)
    assert torch.equal(vp[slots], v)
    # nothing else changed
    rest = torch.ones(kp.shape[0], dtype=torch.bool, device=DEV)
    rest[slots] = False
    assert torch.equal(kp[rest], held[1].flatten(0, 1)[rest])
    assert torch.equal(vp[rest], held[3].flatten(0, 1)[rest])
    assert torch.equal(bk.k_pool[0], held[0]) and torch.equal(bk.v_pool[0], held[2])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_bits_of_rope_then_append(dtype):
    bk, meta, q, k, v = step([(5, 45), (16, 1), (0, 33)], 16, 32, 8, 64, dtype)
    rope = tables(512, 64, 500000.0)
    got = bk.rope_append(0, q, k, v, meta, rope)
    q2, k2 = bk.rope(q, k, meta, rope)
    bk.append_kv(1, k2, v, meta)
    slots = meta.slot_mapping.long()
    assert torch.equal(got, q2)
    assert torch.equal(bk.k_pool[0].flatten(0, 1)[slots], bk.k_pool[1].flatten(0, 1)[slots])
    assert torch.equal(bk.v_pool[0].flatten(0, 1)[slots], bk.v_pool[1].flatten(0, 1)[slots])


def test_layouts_and_outputs():
    bk, meta, q, k, v = step([(5, 45), (0, 3)], 16, 8, 2, 64)
    rope = tables(512, 64)
    want = bk.rope_append(0, q, k, v, meta, rope)
    pool = bk.k_pool[0].clone()
    # contiguous copies, 2-byte aligned views, a transposed layout (copied), fp32 inputs, in place
    for conv in (lambda x: x.contiguous(),
                 lambda x: torch.cat([x.flatten()[:1], x.flatten()])[1:].view(x.shape),
                 lambda x: x.transpose(0, 1).contiguous().transpose(0, 1),
                 lambda x: x.float()):
        bk.k_pool[0].zero_()
        assert torch.equal(bk.rope_append(0, conv(q), conv(k), conv(v), meta, rope), want)
        slots = meta.slot_mapping.long()
        assert torch.equal(bk.k_pool[0].flatten(0, 1)[slots], pool.flatten(0, 1)[slots])
    own = q.contiguous()
    assert bk.rope_append(0, own, k, v, meta, rope, q_out=own) is own and torch.equal(own, want)
    assert bk.rope_append(0, None, k, v, meta, rope) is None
    # on another stream than the tensors were made on
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = bk.rope_append(0, q, k, v, meta, rope)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_nothing_to_append():
    bk, meta, q, k, v = step([(5, 4)])
    empty = slots_meta([])
    out = bk.rope_append(0, q[:0], k[:0], v[:0], empty, tables(64, 64))
    assert out.shape == (0, 8, 64)


def test_bad_slots_and_positions_are_flagged():
    import dataclasses
    bk, meta, q, k, v = step([(5, 45)])
    rope = tables(512, 64)
    slots = meta.slot_mapping.clone()
    slots[3], slots[4] = -1, bk.num_blocks * bk.block_size
    pool = bk.k_pool[0].clone()
    bk.rope_append(0, q, k, v, dataclasses.replace(meta, slot_mapping=slots), rope)
    with pytest.raises(PkvError, match="outside the pool"):
        bk.check_status()
    skipped = meta.slot_mapping[3:5].long()
    assert torch.equal(bk.k_pool[0].flatten(0, 1)[skipped], pool.flatten(0, 1)[skipped])
    pos = meta.positions.clone()
    pos[0], pos[1] = -1, 512
    got = bk.rope_append(0, q, k, v, dataclasses.replace(meta, positions=pos), rope)
    assert torch.equal(got[:2], q[:2])  # left unrotated
    with pytest.raises(PkvError):
        bk.check_status()


def entries(pool):
    """Index entries of whole pages [blocks, page, kv heads, d] (numpy, fp32 steps as defined)."""
    x = pool.float().cpu().numpy()
    lo, hi = x.min(1), x.max(1)
    scale = (np.maximum(abs(lo), abs(hi)).max(-1) * np.float32(1.0 / 127.0)).astype(np.float32)
    safe = np.where(scale > 0, scale, 1)[..., None]
    lo = np.clip(np.floor(lo / safe), -127, 127) * (scale > 0)[..., None]
    hi = np.clip(np.ceil(hi / safe), -127, 127) * (scale > 0)[..., None]
    return np.stack([lo, hi], -2).astype(np.int8), scale


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page,hkv,d", [(16, 8, 64), (16, 2, 128), (8, 3, 40), (5, 1, 33), (32, 9, 256)])
def test_index_of_completed_pages(page, hkv, d, dtype):
    specs = [(0, 3 * page), (page - 1, 1), (page, 1), (2 * page - 1, page + 2), (1, page - 2) if page > 2 else (0, 1)]
    bk, meta, q, k, v = step(specs, page, hkv, hkv, d, dtype)
    index = PageIndex(bk)
    bk.rope_append(1, q, k, v, meta, tables(512, d - d % 2), index=index)
    bk.check_status()
    slots = meta.slot_mapping.cpu().numpy()
    done = sorted({int(s) // page for s in slots if s % page == page - 1})
    codes, scales = entries(bk.k_pool[1])
    assert np.array_equal(index.codes[1].cpu().numpy()[done], codes[done])
    assert np.array_equal(index.scales[1].cpu().numpy()[done], scales[done])
    rest = [b for b in range(bk.num_blocks) if b not in done]
    assert not index.codes[1, rest].any() and not index.scales[1, rest].any() and not index.codes[0].any()
    # the bounds bound every key of the page
    low = index.codes[1, done, :, 0].double() * index.scales[1, done].double()[..., None]
    high = index.codes[1, done, :, 1].double() * index.scales[1, done].double()[..., None]
    keys = bk.k_pool[1][done].double()
    slack = 2.0 ** -22 * keys.abs().amax()
    assert bool((keys >= low[:, None] - slack).all()) and bool((keys <= high[:, None] + slack).all())
    # update alone, and rebuild of every layer, write the same entries
    again = PageIndex(bk)
    again.update(1, meta)
    assert torch.equal(again.codes, index.codes) and torch.equal(again.scales, index.scales)
    again.rebuild(range(bk.num_blocks))
    for l in range(2):
        codes, scales = entries(bk.k_pool[l])
        assert np.array_equal(again.codes[l].cpu().numpy(), codes)
        assert np.array_equal(again.scales[l].cpu().numpy(), scales)


def test_index_of_equal_and_zero_keys():
    bk, *_ = step([(0, 16)])
    bk.k_pool[0].zero_()
    bk.k_pool[1].fill_(-3.0)
    index = PageIndex(bk)
    index.rebuild(torch.arange(bk.num_blocks))
    assert not index.codes[0].any() and not index.scales[0].any()
    assert bool((index.codes[1] == -127).all())
    index.rebuild([])
    with pytest.raises(IndexError):
        index.rebuild([bk.num_blocks])


def test_refusals():
    bk, meta, q, k, v = step([(5, 4)])
    rope = tables(64, 64)
    with pytest.raises(ValueError, match="k has shape"):
        bk.rope_append(0, q, k[:, :1], v, meta, rope)
    with pytest.raises(ValueError, match="v shape"):
        bk.rope_append(0, q, k, v[:2], meta, rope)
    with pytest.raises(ValueError, match="q has shape"):
        bk.rope_append(0, q[:2], k, v, meta, rope)
    with pytest.raises(ValueError, match="slot_mapping has"):
        bk.rope_append(0, q[:2], k[:2], v[:2], meta, rope)
    with pytest.raises(ValueError, match="layer_idx"):
        bk.rope_append(2, q, k, v, meta, rope)
    with pytest.raises(ValueError, match="pair"):
        bk.rope_append(0, q, k, v, meta, rope[0])
    with pytest.raises(ValueError, match="heads of 64"):
        bk.rope_append(0, q, k, v, meta, tables(64, 128))
    with pytest.raises(ValueError, match="float32"):
        bk.rope_append(0, q, k, v, meta, (rope[0].half(), rope[1].half()))
    with pytest.raises(ValueError, match="q_out"):
        bk.rope_append(0, q, k, v, meta, rope, q_out=torch.empty(3, device=DEV))
    with pytest.raises(ValueError, match="overlaps"):
        flat = torch.zeros(q.numel() + 64, dtype=q.dtype, device=DEV)
        bk.rope_append(0, flat[:q.numel()].view(q.shape), k, v, meta, rope, q_out=flat[64:].view(q.shape))
    with pytest.raises(ValueError, match="another backend"):
        other, *_ = step([(5, 4)])
        bk.rope_append(0, q, k, v, meta, rope, index=PageIndex(other))
    with pytest.raises(ValueError, match="fp16, bf16 or fp32"):
        PageIndex(B200PagedBackend(1, 2, 16, 2, 2, 8, device=DEV, dtype=torch.float64))

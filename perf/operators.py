"""
The paged-cache operators and the cases they are measured on.

Three operators over the paged KV pool ``[blocks, page, kv heads, head_dim]``
and the block tables of a step:

* ``append``  the step's q and k rotated at their positions, q returned, k and
  v written to their slots, straight from the slices of the fused qkv
  projection; with ``index`` also the int8 bounds of the pages it completes;
* ``shared``  attention of a batch whose families share their leading pages;
* ``sparse``  attention of each query over the pages that a score of the page
  index selects for it and KV head.

``run`` with ``own`` false computes them from elementary torch operations in
32 bits; with ``own`` true it calls the package. Lengths, page counts and the
families of a case follow from the case alone, values and the scattering of
the pages over the pool from the seed.
"""

import math
import random

import numpy as np
import torch

own = False

PAGE = 16
DEV = "cuda:0"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
INV127 = 1.0 / 127.0


# ---------------------------------------------------------------- the cases
def _append(name, n, q, ctx, dtype="fp16", d=64, hq=32, hkv=8, rot=0, interleaved=False, index=False, lay=1):
    c = dict(op="append", n=n, q=q, ctx=ctx, dtype=dtype, d=d, hq=hq, hkv=hkv, rot=rot or d,
             interleaved=interleaved, index=index, lay=lay)
    return dict(c, name=name) if name else c


def _shared(name, families, n, prefix, tail, q=1, dtype="fp16", hq=32, hkv=8, lay=1):
    c = dict(op="shared", families=families, n=n, prefix=prefix, tail=tail, q=q, dtype=dtype, d=64, hq=hq, hkv=hkv,
             lay=lay)
    return dict(c, name=name) if name else c


def _sparse(name, n, ctx, budget, q=1, dtype="fp16", d=64, hq=32, hkv=8, sink=1, recent=2, lay=1):
    c = dict(op="sparse", n=n, ctx=ctx, budget=budget, q=q, dtype=dtype, d=d, hq=hq, hkv=hkv, sink=sink,
             recent=recent, lay=lay)
    return dict(c, name=name) if name else c


def listed():
    return [
        # a decode step of a few sequences: launch latency
        _append("append decode 8", 8, 1, 2048),
        # one 512-token prompt chunk, the scheduler's chunk size, with the page index kept
        _append("append chunk 512", 1, 512, 1024, dtype="bf16", index=True),
        # a mixed step with wide heads, interleaved pairs and only part of each head rotated
        _append("append mixed 128-wide", 37, 61, 700, d=128, hq=24, hkv=8, rot=96, interleaved=True),
        # the prompts of a full admission wave, index kept
        _append("append prompts 16384", 32, 512, 0, index=True, lay=0),
        # parallel samples of one prompt: latency
        _shared("shared 4 samples", 1, 4, 1024, 64),
        # families of the radix cache, prefixes of 64 to 512 tokens
        _shared("shared 32 families", 32, 256, 512, 768, lay=2),
        # one long system prompt under a full decode batch
        _shared("shared system prompt", 1, 256, 4096, 512, dtype="bf16", lay=3),
        # short question or verification chunks after a shared document
        _shared("shared chunks", 3, 24, 2048, 96, q=12, lay=4),
        # one long document, one sequence: latency
        _sparse("sparse 1 x 32k", 1, 32768, 64),
        # a ragged batch of medium contexts
        _sparse("sparse 32 ragged", 32, 8192, 48, dtype="bf16", lay=2),
        # a full decode batch
        _sparse("sparse 256 x 4k", 256, 4096, 64, lay=3),
        # a few tokens per sequence (verification of drafted tokens), wide heads
        _sparse("sparse drafts 128-wide", 12, 6000, 32, q=5, d=128, hq=16, hkv=4, lay=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "shared", "sparse"])
    dtype = rng.choice(["fp16", "bf16"])
    lay = rng.randrange(1, 1 << 20)
    heads = rng.choice([(32, 8), (32, 4), (16, 8), (8, 8), (8, 1)])
    if op == "append":
        n = _log(rng, 1, 256)
        q = rng.choice([1, _log(rng, 1, max(1, 12000 // n))])
        d = rng.choice([64, 128])
        return _append(None, n, q, _log(rng, 1, 2048), dtype, d, *heads, rot=rng.choice([d, d, d // 2]),
                       interleaved=rng.random() < 0.3, index=rng.random() < 0.5, lay=lay)
    if op == "shared":
        n = _log(rng, 2, 256)
        q = rng.choice([1, 1, _log(rng, 2, 24)])
        n = max(2, min(n, 384 // q))
        families = _log(rng, 1, max(1, n // 2))
        return _shared(None, families, n, _log(rng, 32, 4096), _log(rng, 2, 640) + q, q, dtype, *heads, lay=lay)
    q = rng.choice([1, 1, _log(rng, 2, 8)])
    d = rng.choice([64, 64, 128])
    n = max(1, min(_log(rng, 1, 200), 192 * 64 // (q * d)))
    ctx = _log(rng, 64, min(32768, 700000 * 64 // (n * d)))
    sink, recent = rng.choice([(1, 2), (0, 1), (4, 4)])
    return _sparse(None, n, ctx + q, max(sink + recent, _log(rng, 8, 64)), q, dtype, d, *heads, sink=sink,
                   recent=recent, lay=lay)


# ---------------------------------------------------------------- lengths of a case
def _lens(case):
    """Per sequence: new tokens, tokens after this step, shared leading pages; family sizes."""
    r = random.Random(case["lay"] * 7919 + case["n"])
    n, q = case["n"], case["q"]
    if case["op"] == "append":
        ql = [q if n == 1 or case["lay"] == 0 else r.randint(max(1, q // 2), q) for _ in range(n)]
        kv = [x + (r.randint(0, case["ctx"]) if case["ctx"] else 0) for x in ql]
        return ql, kv, [0] * n, [1] * n
    ql = [r.randint(1, q) for _ in range(n)] if q > 1 else [1] * n
    if case["op"] == "sparse":
        lo = case["ctx"] if n == 1 else max(q, case["ctx"] // 3)
        return ql, [r.randint(lo, case["ctx"]) for _ in range(n)], [0] * n, [1] * n
    f = case["families"]
    sizes = [n // f + (i < n % f) for i in range(f)]
    pre, kv = [], []
    for size in sizes:
        p = max(1, (case["prefix"] if f == 1 else r.randint(max(1, case["prefix"] // 4), case["prefix"])) // PAGE)
        for _ in range(size):
            x = ql[len(kv)]
            kv.append(p * PAGE + r.randint(x, max(x, case["tail"])))
            pre.append(p)
    return ql, kv, pre, sizes


def work(case):
    ql, kv, pre, sizes = _lens(case)
    es, d, hq, hkv = (4 if case["dtype"] == "fp32" else 2), case["d"], case["hq"], case["hkv"]
    T = sum(ql)
    if case["op"] == "append":
        b = T * (2 * (hq + 2 * hkv) * d * es + 12)
        b += len({p for q, k in zip(ql, kv) for p in range(k - q, k)}) * case["rot"] * 4
        if case["index"]:
            done = sum(k // PAGE - (k - q) // PAGE for q, k in zip(ql, kv))
            b += done * hkv * (2 * d + 4)
        return {"bytes": b, "flops": 3 * T * (hq + hkv) * case["rot"]}
    keys = sum((k - q) * q + q * (q + 1) // 2 for q, k in zip(ql, kv))
    b = 2 * T * hq * d * es
    if case["op"] == "shared":
        first = [sum(sizes[:i]) for i in range(len(sizes))]
        rows = sum(k - p * PAGE for k, p in zip(kv, pre)) + sum(pre[i] * PAGE for i in first)
        return {"bytes": b + rows * 2 * hkv * d * es, "flops": 4 * d * hq * keys}
    chosen = cand = flops = 0
    for q, k in zip(ql, kv):
        pages = -(-k // PAGE)
        cand += pages
        chosen += min(pages, case["budget"]) * PAGE
        for p in range(k - q, k):
            own_pages = p // PAGE + 1
            flops += 4 * d * hq * min(own_pages, case["budget"]) * PAGE + 4 * d * hq * own_pages
    return {"bytes": b + cand * hkv * (2 * d + 4) + chosen * 2 * hkv * d * es, "flops": flops}


# ---------------------------------------------------------------- inputs
def _tables(case, seed):
    """Block tables: families share their leading pages; the pages scatter over the pool."""
    ql, kv, pre, sizes = _lens(case)
    total = sum(-(-k // PAGE) - p for k, p in zip(kv, pre)) + sum(
        pre[sum(sizes[:i])] for i in range(len(sizes)))
    ids = np.random.RandomState(seed % (1 << 31)).permutation(total + 8)
    at, i, tables = 0, 0, []
    for size in sizes:
        lead = ids[at:at + pre[i]]
        at += pre[i]
        for _ in range(size):
            more = -(-kv[i] // PAGE) - pre[i]
            tables.append(np.concatenate([lead, ids[at:at + more]]).astype(np.int64))
            at += more
            i += 1
    return ql, kv, pre, sizes, tables, total + 8


def _boxes(k):
    """Index entry of whole pages k [..., page, kv heads, d]: int8 codes [..., kv heads, 2, d] and scales."""
    lo, hi = k.float().amin(-3), k.float().amax(-3)
    scale = torch.maximum(lo.abs(), hi.abs()).amax(-1) * INV127
    safe = scale.unsqueeze(-1) > 0
    low = torch.where(safe, torch.floor(lo / scale.unsqueeze(-1)), 0.0)
    high = torch.where(safe, torch.ceil(hi / scale.unsqueeze(-1)), 0.0)
    return torch.stack([low, high], -2).clamp(-127, 127).to(torch.int8), scale


def prepare(case, seed):
    ql, kv, pre, sizes, tables, blocks = _tables(case, seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    dtype, d, hq, hkv = DTYPES[case["dtype"]], case["d"], case["hq"], case["hkv"]
    n, T = case["n"], sum(ql)
    s = {"case": case, "T": T}

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)

    k_pool = normal(blocks, PAGE, hkv, d, std=0.5 ** 0.5)
    v_pool = normal(blocks, PAGE, hkv, d, std=0.5 ** 0.5)
    if case["op"] == "sparse":  # neighbouring keys are alike: each page has a direction of its own
        k_pool += normal(blocks, 1, hkv, d, std=0.5)
    # the tables as tensors: the page list of each sequence, each new token's sequence, position and slot
    pages = max(len(t) for t in tables)
    table = torch.from_numpy(np.stack([np.pad(t, (0, pages - len(t))) for t in tables])).to(DEV)
    seq_of = np.repeat(np.arange(n), ql)
    pos = np.concatenate([np.arange(k - q, k) for q, k in zip(ql, kv)])
    slots = np.concatenate([t[np.arange(k - q, k) // PAGE] * PAGE + np.arange(k - q, k) % PAGE
                            for t, q, k in zip(tables, ql, kv)])
    s.update(table=table, seq=torch.from_numpy(seq_of).to(DEV), pos=torch.from_numpy(pos).to(DEV))
    if case["op"] == "append":
        qkv = normal(T, (hq + 2 * hkv) * d)  # the projection's output; q, k and v are its slices
        s["q"], s["k"], s["v"] = (x.unflatten(1, (-1, d)) for x in qkv.split([hq * d, hkv * d, hkv * d], 1))
        inv = 500000.0 ** (-torch.arange(0, case["rot"], 2, device=DEV, dtype=torch.float32) / case["rot"])
        ang = torch.arange(max(kv), device=DEV, dtype=torch.float32)[:, None] * inv
        s["rope"] = (torch.cos(ang), torch.sin(ang))
        s["slots"] = torch.from_numpy(slots).to(DEV)
        s["done"] = torch.from_numpy(slots[pos % PAGE == PAGE - 1] // PAGE).to(DEV)
    else:
        s["q"], s["scale"] = normal(T, hq, d), d ** -0.5
    if own:
        import llm_serving_layer_b200 as pkg

        bk = pkg.B200PagedBackend(1, blocks, PAGE, hkv, hq, d, device=DEV, dtype=dtype, validate="device")
        bk.k_pool[0].copy_(k_pool)
        bk.v_pool[0].copy_(v_pool)
        s["backend"] = bk
        s["meta"] = meta = pkg.build_meta([t.tolist() for t in tables], kv, ql, PAGE, device=DEV)
        if case["op"] == "shared":
            s["plan"] = bk.plan_shared(meta, pkg.SharedPrefix(sizes, [pre[sum(sizes[:i])] for i in range(len(sizes))]))
        if case["op"] == "sparse" or case.get("index"):
            s["index"] = pkg.PageIndex(bk)
        if case["op"] == "sparse":
            s["index"].rebuild(range(blocks))
            s["plan"] = bk.plan_sparse(meta, s["index"], budget=case["budget"], sink=case["sink"],
                                       recent=case["recent"])
    else:
        s["k_pool"], s["v_pool"] = k_pool, v_pool
        if case["op"] == "sparse":
            s["codes"], s["scales"] = _boxes(k_pool)
        elif case.get("index"):
            s["codes"] = torch.zeros(blocks, hkv, 2, d, dtype=torch.int8, device=DEV)
            s["scales"] = torch.zeros(blocks, hkv, device=DEV)
    return s


# ---------------------------------------------------------------- plain forms
def _rotate(x, cos, sin, interleaved):
    rot = 2 * cos.shape[-1]
    head = x[..., :rot].float()
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
    else:
        a, b = head[..., :rot // 2], head[..., rot // 2:]
    y = (a * cos - b * sin, a * sin + b * cos)
    y = torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1)
    return torch.cat([y.to(x.dtype), x[..., rot:]], -1)


def _plain_append(s):
    case, (cos, sin) = s["case"], s["rope"]
    cos, sin = cos[s["pos"]][:, None, :], sin[s["pos"]][:, None, :]
    q = _rotate(s["q"], cos, sin, case["interleaved"])
    s["k_pool"].flatten(0, 1)[s["slots"]] = _rotate(s["k"], cos, sin, case["interleaved"])
    s["v_pool"].flatten(0, 1)[s["slots"]] = s["v"]
    out = {"q": q, "k_pool": s["k_pool"], "v_pool": s["v_pool"]}
    if case["index"]:
        s["codes"][s["done"]], s["scales"][s["done"]] = _boxes(s["k_pool"][s["done"]])
        out.update(codes=s["codes"], scales=s["scales"])
    return out


def _softmax_attend(q, k, v, seen, scale):
    """q [T, hkv, g, d], k / v [T, hkv, keys, d], seen [T, 1 or hkv, keys]; fp32."""
    w = (q @ k.transpose(-1, -2)) * scale
    w = w.masked_fill(~seen[:, :, None, :], -math.inf)
    w = torch.exp(w - w.amax(-1, keepdim=True))
    return (w @ v) / w.sum(-1, keepdim=True)


def _plain_shared(s):
    case, table, T = s["case"], s["table"], s["T"]
    q = s["q"].float().unflatten(1, (case["hkv"], -1))
    keys = torch.arange(table.shape[1] * PAGE, device=DEV)
    slots = (table.repeat_interleave(PAGE, 1) * PAGE + keys % PAGE)[s["seq"]]
    k = s["k_pool"].flatten(0, 1)[slots].transpose(1, 2).float()
    v = s["v_pool"].flatten(0, 1)[slots].transpose(1, 2).float()
    seen = keys <= s["pos"][:, None]
    return _softmax_attend(q, k, v, seen[:, None], s["scale"]).reshape(T, case["hq"], case["d"]).to(s["q"].dtype)


def _plain_sparse(s):
    case, T, hkv = s["case"], s["T"], s["case"]["hkv"]
    q = s["q"].float().unflatten(1, (hkv, -1))
    table = s["table"][s["seq"]]  # [T, pages]
    # the score of every page: whole-number products of the int8 query and bounds, then the scales
    qs = q.abs().amax(-1, keepdim=True) * INV127
    q8 = torch.where(qs > 0, torch.round(q / qs), 0.0).clamp(-127, 127)
    code = s["codes"][table].float()  # [T, pages, hkv, 2, d]
    q8 = torch.cat([q8.clamp(max=0), q8.clamp(min=0)], -1)  # times lo where negative, times hi where positive
    dot = q8 @ code.flatten(-2).permute(0, 2, 3, 1)  # [T, hkv, g, pages]
    score = (dot * qs).amax(2) * s["scales"][table].transpose(1, 2)
    at = torch.arange(table.shape[1], device=DEV)
    mine = s["pos"][:, None, None] // PAGE
    score = score.masked_fill((at < case["sink"]) | (at > mine - case["recent"]), math.inf)
    score = score.masked_fill(at > mine, -math.inf).expand(T, hkv, -1)
    score = torch.nn.functional.pad(score, (0, max(0, case["budget"] - score.shape[-1])), value=-math.inf)
    order = score.sort(dim=-1, descending=True, stable=True).indices[..., :case["budget"]].sort(-1).values
    listed_ = order <= mine
    pages = torch.where(listed_, order, -1).to(torch.int32)
    # attention over the listed pages' tokens
    block = table[:, None, :].expand(T, hkv, -1).gather(-1, order.clamp(max=table.shape[1] - 1))
    keys = torch.arange(case["budget"] * PAGE, device=DEV) % PAGE
    slot = block.repeat_interleave(PAGE, -1) * PAGE + keys
    place = order.repeat_interleave(PAGE, -1) * PAGE + keys
    head = torch.arange(hkv, device=DEV)[None, :, None]
    k = s["k_pool"].flatten(0, 1)[slot, head].float()
    v = s["v_pool"].flatten(0, 1)[slot, head].float()
    out = _softmax_attend(q, k, v, place <= s["pos"][:, None, None], s["scale"])
    return {"pages": pages, "out": out.reshape(T, case["hq"], case["d"]).to(s["q"].dtype)}


def run(state):
    s, case = state, state["case"]
    if not own:
        return {"append": _plain_append, "shared": _plain_shared, "sparse": _plain_sparse}[case["op"]](s)
    bk = s["backend"]
    if case["op"] == "append":
        q = bk.rope_append(0, s["q"], s["k"], s["v"], s["meta"], s["rope"], interleaved=case["interleaved"],
                           index=s.get("index"))
        out = {"q": q, "k_pool": bk.k_pool[0], "v_pool": bk.v_pool[0]}
        if case["index"]:
            out.update(codes=s["index"].codes[0], scales=s["index"].scales[0])
        return out
    if case["op"] == "shared":
        return bk.attend_shared(s["q"], 0, s["scale"], s["plan"])
    out, pages = bk.attend_sparse(s["q"], 0, s["scale"], s["plan"])
    return {"pages": pages, "out": out}


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_rope(x, pos, case, cos, sin):
    """x [T, heads, d] as complex numbers turned by the angles of the tables."""
    rot = case["rot"]
    z = x[..., :rot].double()
    z = z.unflatten(-1, (-1, 2)) if case["interleaved"] else z.unflatten(-1, (2, -1)).transpose(-1, -2)
    turn = torch.complex(cos[pos].double(), sin[pos].double())[:, None, :]
    z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
    z = z if case["interleaved"] else z.transpose(-1, -2)
    return torch.cat([z.flatten(-2), x[..., rot:].double()], -1)


def _exact_attend(q, k, v, scale):
    """One query q [hkv, g, d] over k / v [keys, hkv, d]."""
    w = torch.softmax(torch.einsum("hgd,khd->hgk", q, k) * scale, -1)
    return torch.einsum("hgk,khd->hgd", w, v)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    T, hq, hkv, d = s["T"], case["hq"], case["hkv"], case["d"]
    if case["op"] == "append":
        kp, vp = s["k_pool"].double().flatten(0, 1), s["v_pool"].double().flatten(0, 1)
        q = _exact_rope(s["q"], s["pos"], case, *s["rope"])
        kp[s["slots"]] = _exact_rope(s["k"], s["pos"], case, *s["rope"])
        vp[s["slots"]] = s["v"].double()
        out = {"q": q, "k_pool": kp.view(s["k_pool"].shape), "v_pool": vp.view(s["v_pool"].shape)}
        if case["index"]:
            top = torch.zeros(s["scales"].shape, dtype=torch.float64, device=DEV)
            held = out["k_pool"][s["done"]].to(s["k_pool"].dtype).double()  # the bounds are of the keys as held
            top[s["done"]] = held.abs().amax((1, 3)) / 127
            out.update(codes=None, scales=top)
        return out
    pos, seq = s["pos"].tolist(), s["seq"].tolist()
    out = torch.empty(T, hkv, hq // hkv, d, dtype=torch.float64, device=DEV)
    kp, vp = s["k_pool"].flatten(0, 1), s["v_pool"].flatten(0, 1)
    if case["op"] == "shared":
        for t in range(T):
            at = torch.arange(pos[t] + 1, device=DEV)
            at = s["table"][seq[t]][at // PAGE] * PAGE + at % PAGE
            out[t] = _exact_attend(s["q"][t].double().view(hkv, -1, d), kp[at].double(), vp[at].double(), s["scale"])
        return out.view(T, hq, d)
    # sparse: scores from whole numbers, the two scales applied as 32-bit products, on the host
    codes, scales = s["codes"].cpu().numpy().astype(np.int64), s["scales"].cpu().numpy()
    table, q = s["table"].cpu().numpy(), s["q"].float().cpu().numpy().reshape(T, hkv, -1, d)
    pages = np.full((T, hkv, case["budget"]), -1, np.int32)
    for t in range(T):
        mine = pos[t] // PAGE
        ids = table[seq[t]][:mine + 1]
        for h in range(hkv):
            qs = np.abs(q[t, h]).max(-1) * np.float32(INV127)
            q8 = np.clip(np.rint(q[t, h] / np.where(qs > 0, qs, 1)[:, None]), -127, 127).astype(np.int64)
            each = np.maximum(q8[:, None] * codes[ids, h, 0], q8[:, None] * codes[ids, h, 1]).sum(-1)
            score = (each.astype(np.float32) * qs[:, None]).max(0) * scales[ids, h]
            kept = [p for p in range(mine + 1) if p < case["sink"] or p > mine - case["recent"]]
            rest = sorted(set(range(mine + 1)) - set(kept), key=lambda p: (-score[p], p))
            chosen = sorted(kept[:case["budget"]] + rest[:max(0, case["budget"] - len(kept))])
            pages[t, h, :len(chosen)] = chosen
            at = (np.asarray(chosen)[:, None] * PAGE + np.arange(PAGE)).ravel()
            at = at[at <= pos[t]]
            at = torch.from_numpy(table[seq[t]][at // PAGE] * PAGE + at % PAGE).to(DEV)
            w = torch.softmax(s["q"][t].double().view(hkv, -1, d)[h] @ kp[at, h].double().T * s["scale"], -1)
            out[t, h] = w @ vp[at, h].double()
    return {"pages": torch.from_numpy(pages), "out": out.view(T, hq, d)}

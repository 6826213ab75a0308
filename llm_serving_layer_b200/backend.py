"""
B200PagedBackend — the paged-KV attention backend on hand-written sm_100a kernels.

A drop-in for the reference's ``PagedTorchBackend``
(``serving/backends/paged_torch.py:71-509``) and ``FlashInferBackend``
(``serving/backends/flashinfer_backend.py:233-734``): the same constructor, the
same ``append_kv`` / ``attend`` / ``copy_block`` methods, the same accounting
helpers, the same validation errors (``ValueError`` for shapes, layer index
and page-table inconsistencies; ``IndexError`` for ``copy_block`` ranges), and
``k_pool`` / ``v_pool`` as per-layer ``[num_blocks, block_size, n_kv_heads,
head_dim]`` tensors — here views into ONE allocation laid out
``[num_layers][K|V][num_blocks][block_size][n_kv_heads][head_dim]`` so that the
kernels address every layer from one base pointer and one TMA descriptor.

Every operation launches this package's CUDA kernels through ``libpkv.so``
(C ABI, ``include/pkv.h``) on ``torch.cuda.current_stream()``; there is no
torch or CPU fallback, and construction fails on a non-CUDA device.
"""

from __future__ import annotations

import ctypes
from types import SimpleNamespace
from typing import Any, Sequence

import torch

from . import _native as N

__all__ = ["B200PagedBackend", "SharedPlan", "SparsePlan"]


class SharedPlan:
    """One step of ``attend_shared``: made by ``B200PagedBackend.plan_shared``,
    used by every layer of the step. Holds the step's tables and a workspace of
    its own (``workspace`` may be passed on to the next step's plan)."""

    __slots__ = ("backend", "meta", "n_tokens", "batch", "batch_ref", "tensors", "workspace", "ws_ptr", "ws_bytes")


class SparsePlan:
    """One step of ``attend_sparse``: made by ``B200PagedBackend.plan_sparse``,
    used by every layer of the step."""

    __slots__ = ("backend", "index", "budget", "sink", "recent", "max_pages", "n_tokens", "batch", "batch_ref",
                 "tensors", "rows_ptr")


class B200PagedBackend:
    """Paged KV storage plus attention on B200 kernels.

    ``validate``:
      * ``"host"`` (default) — once per ``BatchMeta`` (cached by identity, as
        ``FlashInferBackend._ensure_planned`` caches its plan) the page table is
        read back and checked on the host, raising the reference's
        ``ValueError``s before any kernel runs; ``is_prefill`` is cross-checked
        against ``query_lens``.
      * ``"device"`` — no host round trip: kernels check the page table and OR
        violations into a device status word; ``check_status()`` raises them.
    """

    def __init__(
        self,
        num_layers: int,
        num_blocks: int,
        block_size: int,
        n_kv_heads: int,
        n_heads: int,
        head_dim: int,
        device: str | torch.device = "cuda:0",
        dtype: torch.dtype = torch.float16,
        *,
        validate: str = "host",
    ):
        if n_heads % n_kv_heads != 0:
            raise ValueError(
                f"n_heads={n_heads} must be divisible by n_kv_heads={n_kv_heads}; "
                "GQA maps query head h to KV head h // (n_heads // n_kv_heads)."
            )
        for name, val in (
            ("num_layers", num_layers), ("num_blocks", num_blocks), ("block_size", block_size),
            ("n_kv_heads", n_kv_heads), ("n_heads", n_heads), ("head_dim", head_dim),
        ):
            if val <= 0:
                raise ValueError(f"{name} must be positive, got {val}")
        if validate not in ("host", "device"):
            raise ValueError(f"validate must be 'host' or 'device', got {validate!r}")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError(
                f"B200PagedBackend requires a CUDA device, got {self.device}; it has no CPU path"
            )
        if dtype not in N.DTYPE_CODE:
            raise ValueError(f"unsupported pool dtype {dtype}")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self._lib = N.lib()

        self.num_layers = num_layers
        self.num_blocks = num_blocks
        self.block_size = block_size
        self.n_kv_heads = n_kv_heads
        self.n_heads = n_heads
        self.head_dim = head_dim
        self.dtype = dtype
        self.groups = n_heads // n_kv_heads
        self.validate = validate

        self._pool = torch.zeros(
            (num_layers, 2, num_blocks, block_size, n_kv_heads, head_dim), dtype=dtype, device=self.device
        )
        self.k_pool: list[torch.Tensor] = [self._pool[l, 0] for l in range(num_layers)]
        self.v_pool: list[torch.Tensor] = [self._pool[l, 1] for l in range(num_layers)]
        self._desc = N.PoolDesc(
            self._pool.data_ptr(), num_blocks, num_layers, block_size, n_kv_heads, head_dim,
            N.DTYPE_CODE[dtype], 0,
        )
        self._pdesc = ctypes.byref(self._desc)
        self._status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._status_ptr = self._status.data_ptr()
        self._dev_index = self.device.index if self.device.index is not None else torch.cuda.current_device()
        self._slots_meta: Any = None  # the meta whose int32 slot map is cached in _slots
        self._slots: torch.Tensor | None = None
        self._pos_meta: Any = None  # the meta whose int64 device positions are cached in _pos
        self._pos: torch.Tensor | None = None
        self._ws: torch.Tensor | None = None
        self._indexes: list[Any] = []  # weak references to the PageIndex objects of this pool
        # per-step state, keyed by BatchMeta identity (a strong reference keeps
        # the id from being recycled while it is cached)
        self._meta: Any = None
        self._meta_state: dict[str, Any] = {}
        self.n_plans = 0
        self.n_runs = 0
        self.last_kernel: str | None = None  # "decode" | "prefill" | "generic": kernel of the last attend

    # -- accounting (paged_torch.py:139-177) ----------------------------------

    def zeros_like_pool(self) -> torch.Tensor:
        return torch.zeros(
            (self.num_blocks, self.block_size, self.n_kv_heads, self.head_dim),
            dtype=self.dtype, device=self.device,
        )

    def pool_bytes(self) -> int:
        return self._pool.numel() * self._pool.element_size()

    def block_bytes(self) -> int:
        return self.pool_bytes() // self.num_blocks

    def workspace_bytes(self) -> int:
        return 0 if self._ws is None else self._ws.numel()

    def tokens_capacity(self) -> int:
        return self.num_blocks * self.block_size

    @staticmethod
    def estimate_pool_bytes(num_layers: int, num_blocks: int, block_size: int, n_kv_heads: int,
                            head_dim: int, dtype: torch.dtype = torch.float16) -> int:
        elem = torch.empty((), dtype=dtype).element_size()
        return num_layers * 2 * num_blocks * block_size * n_kv_heads * head_dim * elem

    # -- write path ------------------------------------------------------------

    def copy_block(self, src: int, dst: int) -> None:
        """Duplicate one block, every layer, K and V (copy-on-write;
        ``paged_torch.py:181-207``). ``IndexError`` out of range; no-op if equal."""
        src, dst = int(src), int(dst)
        if not (0 <= src < self.num_blocks and 0 <= dst < self.num_blocks):
            raise IndexError(f"copy_block({src} -> {dst}) outside [0, {self.num_blocks})")
        if src == dst:
            return
        N.check(self._lib.pkv_copy_block(self._pdesc, src, dst, N.stream_ptr(self.device)),
                "copy_block", IndexError)
        if self._indexes:
            self._reindex_blocks(torch.full((1,), dst, dtype=torch.int32, device=self.device))

    def copy_blocks(self, src: Sequence[int] | torch.Tensor, dst: Sequence[int] | torch.Tensor) -> None:
        """Batched ``copy_block``: all pairs, all layers, one launch. The
        destination set must not intersect the source set (a chain a->b->c would
        depend on order); pairs with src == dst are skipped."""
        s = torch.as_tensor(src, dtype=torch.int32).flatten()
        d = torch.as_tensor(dst, dtype=torch.int32).flatten()
        if s.shape != d.shape:
            raise ValueError(f"{s.numel()} sources but {d.numel()} destinations")
        if s.numel() == 0:
            return
        hs, hd = s.cpu(), d.cpu()
        lo = int(torch.minimum(hs.min(), hd.min()))
        hi = int(torch.maximum(hs.max(), hd.max()))
        if lo < 0 or hi >= self.num_blocks:
            raise IndexError(f"copy_blocks ids outside [0, {self.num_blocks})")
        moving = hs != hd
        if bool(torch.isin(hd[moving], hs[moving]).any()):
            raise ValueError("copy_blocks: a destination is also a source; issue the pairs in order")
        if len(set(hd[moving].tolist())) != int(moving.sum()):
            raise ValueError("copy_blocks: duplicate destination block")
        s, d = s.to(self.device), d.to(self.device)
        N.check(self._lib.pkv_copy_blocks(self._pdesc, s.data_ptr(), d.data_ptr(), s.numel(),
                                          self._status.data_ptr(), N.stream_ptr(self.device)),
                "copy_blocks")
        if self._indexes:
            self._reindex_blocks(d)

    def append_kv(self, layer_idx: int, k: torch.Tensor, v: torch.Tensor, meta: Any) -> None:
        """Scatter this step's K/V into the pool at ``meta.slot_mapping``
        (``paged_torch.py:209-276``). Idempotent."""
        k, v, slots, tokens = self._append_args(layer_idx, k, v, meta)
        if tokens == 0:
            return
        N.check(self._lib.pkv_append_kv(self._pdesc, layer_idx, k.data_ptr(), v.data_ptr(),
                                        slots.data_ptr(), tokens, self._status_ptr,
                                        N.raw_stream(self._dev_index)), "append_kv")
        if self._indexes:
            self._reindex_step(layer_idx, slots)

    def append_attend(self, layer_idx: int, k: torch.Tensor, v: torch.Tensor, q: torch.Tensor,
                      scale: float, meta: Any, *, out: torch.Tensor | None = None,
                      rope: tuple[torch.Tensor, torch.Tensor] | None = None) -> torch.Tensor:
        """``append_kv(layer_idx, k, v, meta)`` then ``attend(q, layer_idx, scale,
        meta)`` in one call, with the same checks, errors and results. A decode
        step is ONE kernel launch: the decode kernel writes each sequence's new
        K/V row to its slot and attends over it (no reference counterpart; the
        engine makes the two calls, ``docs/ARCHITECTURE.md:167-172``).

        ``rope=(cos, sin)``: q and k are given before the rotary embedding, which
        is applied at ``meta.positions`` with these fp32 tables
        ``[max_pos, head_dim // 2]`` (see ``rope``); the pool receives the
        rotated K and the result is that of ``rope`` followed by this call, bit
        for bit. For a decode step the rotation happens inside the single
        launch; other steps run ``rope`` first (one launch for q and k)."""
        if rope is not None:
            return self._append_attend_rope(layer_idx, k, v, q, scale, meta, out, rope)
        k, v, slots, tokens = self._append_args(layer_idx, k, v, meta)
        if q.shape != (tokens, self.n_heads, self.head_dim):
            raise ValueError(
                f"q has shape {tuple(q.shape)}, expected ({tokens}, {self.n_heads}, {self.head_dim})"
            )
        st = self._step_state(meta)
        if st["n_tokens"] != tokens:
            raise ValueError(f"meta describes {st['n_tokens']} tokens but q has {tokens}")
        q = self._own(q, self.dtype)
        out = self._out(q, out)
        if tokens == 0:
            return out
        self.n_runs += 1
        self.last_kernel = st["kernel"]
        N.check(self._lib.pkv_append_attend_planned(
            self._pdesc, layer_idx, self.n_heads, k.data_ptr(), v.data_ptr(), slots.data_ptr(), q.data_ptr(),
            out.data_ptr(), float(scale), st["batch_ref"], st["hint"], st["ws_ptr"], st["ws_bytes"],
            N.raw_stream(self._dev_index)), "append_attend")
        if self._indexes:
            self._reindex_step(layer_idx, slots)
        return out

    def _append_attend_rope(self, layer_idx, k, v, q, scale, meta, out, rope) -> torch.Tensor:
        cos, sin, pos = self._rope_args(rope, meta)
        k, v, slots, tokens = self._append_args(layer_idx, k, v, meta)
        if pos.shape[0] != tokens:
            raise ValueError(f"meta.positions has {pos.shape[0]} entries but {tokens} tokens were supplied")
        if q.shape != (tokens, self.n_heads, self.head_dim):
            raise ValueError(
                f"q has shape {tuple(q.shape)}, expected ({tokens}, {self.n_heads}, {self.head_dim})"
            )
        st = self._step_state(meta)
        if st["n_tokens"] != tokens:
            raise ValueError(f"meta describes {st['n_tokens']} tokens but q has {tokens}")
        q = self._own(q, self.dtype)
        out = self._out(q, out)
        if tokens == 0:
            return out
        rc = self._lib.pkv_append_attend_rope_planned(
            self._pdesc, layer_idx, self.n_heads, k.data_ptr(), v.data_ptr(), slots.data_ptr(), q.data_ptr(),
            out.data_ptr(), float(scale), st["batch_ref"], st["hint"], st["ws_ptr"], st["ws_bytes"],
            pos.data_ptr(), cos.data_ptr(), sin.data_ptr(), cos.shape[0], N.raw_stream(self._dev_index))
        if rc == N.PKV_ERR_UNSUPPORTED:  # not a single-launch decode step: rotate, then the plain call
            q, k = self.rope(q, k, meta, rope)
            return self.append_attend(layer_idx, k, v, q, scale, meta, out=out)
        N.check(rc, "append_attend")
        self.n_runs += 1
        self.last_kernel = st["kernel"]
        if self._indexes:
            self._reindex_step(layer_idx, slots)
        return out

    def rope(self, q: torch.Tensor | None, k: torch.Tensor | None, meta: Any,
             rope: tuple[torch.Tensor, torch.Tensor]) -> tuple[torch.Tensor | None, torch.Tensor | None]:
        """Rotary position embedding of q ``(T, n_heads, head_dim)`` and k
        ``(T, n_kv_heads, head_dim)`` at ``meta.positions``, returned as new
        tensors in the pool dtype (either input may be None). ``rope = (cos,
        sin)``: fp32 tables ``[max_pos, head_dim // 2]`` on this device; pair
        (i, i + head_dim/2) of each head of token t is rotated by
        cos/sin[positions[t], i] — ``a*cos - b*sin, a*sin + b*cos`` with each
        product rounded to fp32, then rounded to the pool dtype, the bits of
        that formula evaluated elementwise in fp32. One kernel launch
        (``pkv_rope``). A position outside the tables raises on the next
        ``check_status`` (and leaves its token unrotated)."""
        cos, sin, pos = self._rope_args(rope, meta)
        T = int(pos.shape[0])
        qo = ko = None
        args = []
        for x, heads, name in ((q, self.n_heads, "q"), (k, self.n_kv_heads, "k")):
            if x is None:
                args.append((None, None, 0))
                continue
            if x.shape != (T, heads, self.head_dim):
                raise ValueError(f"{name} has shape {tuple(x.shape)}, expected ({T}, {heads}, {self.head_dim})")
            x = self._own(x, self.dtype)
            y = torch.empty_like(x)
            args.append((x, y, heads))
        (xq, qo, hq), (xk, ko, hk) = args
        N.check(self._lib.pkv_rope(
            N.DTYPE_CODE[self.dtype], N.ptr(xq), N.ptr(qo), hq, N.ptr(xk), N.ptr(ko), hk, T, self.head_dim,
            pos.data_ptr(), cos.data_ptr(), sin.data_ptr(), cos.shape[0], self._status_ptr,
            N.raw_stream(self._dev_index)), "rope")
        return qo, ko

    def rope_append(self, layer_idx: int, q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, meta: Any,
                    rope: tuple[torch.Tensor, torch.Tensor], *, interleaved: bool = False, index: Any = None,
                    q_out: torch.Tensor | None = None) -> torch.Tensor | None:
        """Rotates q ``(T, n_heads, head_dim)`` and k ``(T, n_kv_heads, head_dim)``
        at ``meta.positions`` and appends the rotated k and v at
        ``meta.slot_mapping``, in one launch for any step; returns the rotated q
        (``q_out``, which may be q itself but not overlap k or v, or a new
        tensor; None when q is None). q, k and v may be
        slices of the fused projection: any stride between tokens, each token's
        heads contiguous (other layouts are copied first).

        ``rope = (cos, sin)``: fp32 ``[max_pos, rotary_dim // 2]`` on this
        device, ``rotary_dim <= head_dim``; the dims after rotary_dim pass
        through. Pair (i, i + rotary_dim // 2) is turned, or (2i, 2i + 1) when
        ``interleaved``. Same bits as ``rope`` followed by ``append_kv``.
        The entries of the pages this step completes are written too, in
        ``index`` (a ``PageIndex`` of this backend) by the same call and in the
        backend's other indexes after it. fp16, bf16 or fp32 pools."""
        # the checks of every call in their cheapest form; the tables' refusal is worded by a helper
        dev, D, Hk = self._dev_index, self.head_dim, self.n_kv_heads
        try:
            cos, sin = rope
            rows, half = shape = cos.shape
            ok = (half > 0 and rows > 0 and sin.shape == shape and cos.dtype is sin.dtype is torch.float32
                  and cos.get_device() == sin.get_device() == dev and cos.is_contiguous() and sin.is_contiguous())
        except (TypeError, ValueError, AttributeError):
            ok = False
        if not ok:
            self._refuse_rope_tables(rope)
        if 2 * half > D:
            raise ValueError(f"the rope tables turn {2 * half} dims of heads of {D}")
        if layer_idx is None or not 0 <= layer_idx < self.num_layers:
            self._check_layer(layer_idx)
        slots, pos = meta.slot_mapping, meta.positions
        if slots is None or pos is None:
            raise ValueError("rope_append requires meta.slot_mapping and meta.positions")
        shape = k.shape
        tokens = shape[0]
        if shape != (tokens, Hk, D):
            raise ValueError(f"k has shape {tuple(shape)}, expected ({tokens}, {Hk}, {D})")
        if v.shape != shape:
            raise ValueError(f"v shape {tuple(v.shape)} != k shape {tuple(shape)}")
        if slots.shape != (tokens,) or pos.shape != (tokens,):
            raise ValueError(f"slot_mapping has {slots.shape[0]} entries and positions {pos.shape[0]} but {tokens} "
                             "tokens were supplied")
        if index is not None and index.backend is not self:
            raise ValueError("index belongs to another backend")
        dt, row = self.dtype, Hk * D
        ks, vs = k.stride(), v.stride()
        if not (k.dtype is v.dtype is dt and k.get_device() == v.get_device() == dev and ks[1] == vs[1] == D
                and ks[2] == vs[2] == 1 and ks[0] >= row and vs[0] >= row):
            (k, ks), (v, vs) = self._rows(k, row), self._rows(v, row)
        q_ptr = qo_ptr = None
        q_stride = heads = 0
        if q is not None:
            heads = self.n_heads
            if q.shape != (tokens, heads, D):
                raise ValueError(f"q has shape {tuple(q.shape)}, expected ({tokens}, {heads}, {D})")
            qs = q.stride()
            if not (q.dtype is dt and q.get_device() == dev and qs[1] == D and qs[2] == 1 and qs[0] >= heads * D):
                q, qs = self._rows(q, heads * D)
            q_stride = qs[0]
            if q_out is None:
                q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
            elif (q_out.shape != q.shape or q_out.dtype != dt or q_out.get_device() != dev
                  or not q_out.is_contiguous()):
                raise ValueError(f"q_out must be a contiguous {tuple(q.shape)} {dt} tensor on {self.device}")
            elif _overlap(q_out, q) and not (q_out.data_ptr() == q.data_ptr() and q.is_contiguous()):
                raise ValueError("q_out overlaps q without being q")
            elif _overlap(q_out, k) or _overlap(q_out, v):
                raise ValueError("q_out overlaps k or v (a row may be read after q_out has been written)")
            q_ptr, qo_ptr = q.data_ptr(), q_out.data_ptr()
        elif q_out is not None:
            raise ValueError("q_out given without q")
        if not tokens:
            return q_out
        if not (slots.dtype is torch.int32 and pos.dtype is torch.int64
                and slots.get_device() == pos.get_device() == dev and slots.is_contiguous() and pos.is_contiguous()):
            slots, pos = self._i32(slots), self._own(pos, torch.int64)
        rc = self._lib.pkv_rope_append(
            self._pdesc, layer_idx, q_ptr, q_stride, qo_ptr, heads, k.data_ptr(), ks[0], v.data_ptr(), vs[0],
            slots.data_ptr(), pos.data_ptr(), tokens, cos.data_ptr(), sin.data_ptr(), rows, 2 * half, interleaved,
            None if index is None else index._pdesc, self._status_ptr, N.raw_stream(self._dev_index))
        if rc:
            N.check(rc, "rope_append")
        if self._indexes:
            self._reindex_step(layer_idx, slots, index)
        return q_out

    def _reindex_step(self, layer_idx: int, slots: torch.Tensor, done: Any = None) -> None:
        """The pages whose last slot is among ``slots`` (int32, on this device),
        in every index of this pool but ``done``."""
        for ref in self._indexes:
            index = ref()
            if index is not None and index is not done:
                index._write(layer_idx, slots)

    def _reindex_blocks(self, ids: torch.Tensor) -> None:
        """Whole blocks (ids int32, on this device), every layer, in every index of this pool."""
        for ref in self._indexes:
            index = ref()
            if index is not None:
                index._write(-1, ids)

    def _refuse_rope_tables(self, rope):
        try:
            cos, sin = rope
        except (TypeError, ValueError):
            raise ValueError("rope must be a (cos, sin) pair of tensors") from None
        raise ValueError(f"rope cos and sin must be contiguous float32 [max_pos, rotary_dim // 2] tensors of one shape "
                         f"on {self.device}")

    def _rows(self, t: torch.Tensor, row: int) -> tuple[torch.Tensor, tuple[int, ...]]:
        """t ``(T, heads, head_dim)`` on this device in the pool dtype with each
        token's ``row`` elements contiguous (no copy for slices of a fused
        projection), and its strides."""
        st = t.stride()
        if t.dtype is self.dtype and t.get_device() == self._dev_index and st[2] == 1 and st[0] >= row \
                and (st[1] == self.head_dim or row == self.head_dim):
            return t, st
        return t.to(device=self.device, dtype=self.dtype).contiguous(), (row,)

    def _rope_args(self, rope, meta):
        try:
            cos, sin = rope
        except (TypeError, ValueError):
            raise ValueError("rope must be a (cos, sin) pair of tensors") from None
        half = self.head_dim // 2
        for t, name in ((cos, "cos"), (sin, "sin")):
            if (not isinstance(t, torch.Tensor) or t.dim() != 2 or t.shape[1] != half or t.shape[0] < 1
                    or t.dtype != torch.float32 or not t.is_cuda or t.get_device() != self._dev_index
                    or not t.is_contiguous() or t.data_ptr() % 16):
                raise ValueError(
                    f"rope {name} must be a contiguous 16-byte aligned float32 [max_pos, {half}] tensor on "
                    f"{self.device}")
        if cos.shape != sin.shape:
            raise ValueError(f"rope cos {tuple(cos.shape)} and sin {tuple(sin.shape)} differ in shape")
        if getattr(meta, "positions", None) is None:
            raise ValueError("the rotary embedding needs meta.positions")
        if self._pos_meta is not meta:  # the int64 device positions, once per meta
            self._pos = self._own(meta.positions, torch.int64)
            if self._pos.dim() != 1:
                raise ValueError("meta.positions must be one-dimensional")
            self._pos_meta = meta
        return cos, sin, self._pos

    def _append_args(self, layer_idx: int, k: torch.Tensor, v: torch.Tensor, meta: Any):
        self._check_layer(layer_idx)
        if getattr(meta, "slot_mapping", None) is None:
            raise ValueError(
                "B200PagedBackend.append_kv requires meta.slot_mapping (the flat "
                "per-token physical slot)."
            )
        tokens = k.shape[0]
        if k.shape != (tokens, self.n_kv_heads, self.head_dim):
            raise ValueError(
                f"k has shape {tuple(k.shape)}, expected ({tokens}, {self.n_kv_heads}, {self.head_dim})"
            )
        if v.shape != k.shape:
            raise ValueError(f"v shape {tuple(v.shape)} != k shape {tuple(k.shape)}")
        if meta.slot_mapping.shape[0] != tokens:
            raise ValueError(
                f"slot_mapping has {meta.slot_mapping.shape[0]} entries but {tokens} tokens were supplied"
            )
        k = self._own(k, self.dtype)
        v = self._own(v, self.dtype)
        if not tokens:
            return k, v, None, tokens
        if self._slots_meta is not meta:  # the int32 device slot map, once per meta
            self._slots = self._i32(meta.slot_mapping)
            self._slots_meta = meta
        return k, v, self._slots, tokens

    # -- read path -------------------------------------------------------------

    def attend(self, q: torch.Tensor, layer_idx: int, scale: float, meta: Any, *,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention over each sequence's full KV history including this step's
        append (``paged_torch.py:280-485``): GQA ``h // groups``, bottom-right
        causal mask, pages read in listed order, the unwritten tail of the last
        page never read. Returns ``(tokens, n_heads, head_dim)`` in the pool dtype:
        a new tensor, or ``out`` (an optional extension of the reference's
        signature: a contiguous tensor of that shape and dtype on this device,
        written in place)."""
        self._check_layer(layer_idx)
        tokens = q.shape[0]
        if q.shape != (tokens, self.n_heads, self.head_dim):
            raise ValueError(
                f"q has shape {tuple(q.shape)}, expected ({tokens}, {self.n_heads}, {self.head_dim})"
            )
        st = self._step_state(meta)
        if st["n_tokens"] != tokens:
            raise ValueError(f"meta describes {st['n_tokens']} tokens but q has {tokens}")
        q = self._own(q, self.dtype)
        out = self._out(q, out)
        if tokens == 0:
            return out
        self.n_runs += 1
        self.last_kernel = st["kernel"]
        N.check(self._lib.pkv_attend_planned(
            self._pdesc, layer_idx, self.n_heads, q.data_ptr(), out.data_ptr(), float(scale),
            st["batch_ref"], st["hint"], st["ws_ptr"], st["ws_bytes"],
            N.raw_stream(self._dev_index)), "attend")
        return out

    # -- attention of a batch that shares leading pages ---------------------------
    def plan_shared(self, meta: Any, shared: Any, *, workspace: torch.Tensor | None = None) -> SharedPlan:
        """Prepare a step whose sequences come in families that share leading
        pages (``shared``: a ``SharedPrefix``). The returned plan serves every
        layer's ``attend_shared``; its tables are copies, so ``meta`` may be
        reused. ``workspace``: a finished plan's, taken over when large enough.
        A family whose page lists disagree, or whose shared pages reach past the
        tokens before the step, raises ``ValueError`` with ``validate="host"``;
        with ``"device"`` it is computed without sharing and recorded for
        ``check_status``."""
        n = int(meta.query_lens.shape[0])
        if shared.n_seqs != n:
            raise ValueError(f"the groups hold {shared.n_seqs} sequences but the batch has {n}")
        plan = SharedPlan()
        self._plan_batch(plan, meta)
        plan.meta = None
        seen = None
        if self.validate == "host":
            seen = self._host_validate(meta, n, int(meta.kv_indices.shape[0]))
            self._validate_shared(meta, shared)
        bounds = [0]
        for size in shared.group_sizes:
            bounds.append(bounds[-1] + size)
        groups = torch.tensor(bounds + shared.prefix_pages, dtype=torch.int32).to(self.device)
        plan.tensors["groups"] = groups
        b = plan.batch
        need = int(self._lib.pkv_shared_workspace_size(self._pdesc, self.n_heads, n, plan.n_tokens, b.total_pages))
        if need == 0:  # other geometries: every sequence by itself, in attend
            if self.validate == "device":
                N.check(self._lib.pkv_check_shared(
                    self._pdesc, plan.batch_ref, len(shared.group_sizes), groups.data_ptr(),
                    groups.data_ptr() + 4 * len(bounds), N.stream_ptr(self.device)), "plan_shared")
            plan.meta = self._plan_meta(plan, meta, seen)
            plan.workspace, plan.ws_ptr, plan.ws_bytes = None, None, 0
            return plan
        if (workspace is None or workspace.dtype != torch.uint8 or workspace.numel() < need
                or workspace.device != self.device or not workspace.is_contiguous()):
            workspace = torch.empty(need, dtype=torch.uint8, device=self.device)
        plan.workspace, plan.ws_ptr, plan.ws_bytes = workspace, workspace.data_ptr(), workspace.numel()
        N.check(self._lib.pkv_plan_shared(
            self._pdesc, self.n_heads, plan.batch_ref, len(shared.group_sizes), groups.data_ptr(),
            groups.data_ptr() + 4 * len(bounds), plan.ws_ptr, plan.ws_bytes, N.stream_ptr(self.device)), "plan_shared")
        return plan

    def _plan_meta(self, plan: SharedPlan, meta: Any, seen: tuple[bool, int] | None) -> SimpleNamespace:
        """What ``attend`` reads of a step, made of the plan's own tables: an
        object that no other step has (``attend`` knows its steps by identity).
        ``seen``: the result of the host validation that was made, if any."""
        t = plan.tensors
        own = SimpleNamespace(
            query_lens=t["cu"][1:] - t["cu"][:-1], cu_query_lens=t["cu"], kv_lens=t["kl"], kv_indptr=t["ip"],
            kv_indices=t["ix"], kv_last_page_len=t["lp"], slot_mapping=None,
            positions=torch.empty(plan.n_tokens, dtype=torch.int64, device="meta"))  # counted, not read
        if seen is not None:
            decode, hint = seen
            own.is_prefill, own.max_query_len, own.min_query_len = not decode, 1 if decode else 2, 2 if hint == 2 else 1
            own.checked_blocks = self.num_blocks
            return own
        for name in ("is_prefill", "max_query_len", "min_query_len"):
            if hasattr(meta, name):
                setattr(own, name, getattr(meta, name))
        return own

    def attend_shared(self, q: torch.Tensor, layer_idx: int, scale: float, plan: SharedPlan, *,
                      out: torch.Tensor | None = None) -> torch.Tensor:
        """``attend`` for a step planned by ``plan_shared``: same result (to
        rounding), the pages a family shares read once for all its sequences:
        faster where prefixes are long, families large or new tokens several,
        up to 1.4 times slower for pairs and for prefixes of a few pages. Rows
        of a sequence with inconsistent tables are zeros. A step with more than
        16384 new tokens in families (8192 of sequences with several) is computed
        without sharing.
        Geometries outside the tensor-core kernels' (fp16 / bf16, head_dim 64,
        16-token pages, up to 8 KV heads, 1/2/4/8 query heads per KV head) run
        ``attend`` itself."""
        if plan.backend is not self:  # its page ids were checked against that pool
            raise ValueError("the plan belongs to another backend")
        if plan.meta is not None:
            return self.attend(q, layer_idx, scale, plan.meta, out=out)
        if layer_idx is None or not 0 <= layer_idx < self.num_layers:
            self._check_layer(layer_idx)
        q = self._query(q, plan.n_tokens)
        out = torch.empty_like(q) if out is None else self._out(q, out)
        if not plan.n_tokens:
            return out
        rc = self._lib.pkv_attend_shared_planned(
            self._pdesc, layer_idx, self.n_heads, q.data_ptr(), out.data_ptr(), scale, plan.batch_ref,
            plan.ws_ptr, plan.ws_bytes, N.raw_stream(self._dev_index))
        if rc:
            N.check(rc, "attend_shared")
        self.n_runs += 1
        self.last_kernel = "shared"
        return out

    def _validate_shared(self, meta: Any, shared: Any) -> None:
        ip, ix = meta.kv_indptr.tolist(), meta.kv_indices.tolist()
        ql, lp = meta.query_lens.tolist(), meta.kv_last_page_len.tolist()
        s = 0
        for g, (size, pages) in enumerate(zip(shared.group_sizes, shared.prefix_pages)):
            lead = ix[ip[s]:ip[s] + pages]
            for i in range(s, s + size) if pages else ():
                kv = (ip[i + 1] - ip[i] - 1) * self.block_size + lp[i]
                if pages * self.block_size > kv - ql[i]:
                    raise ValueError(f"group {g}: {pages} shared pages reach past the {kv - ql[i]} tokens sequence "
                                     f"{i} held before this step")
                if ix[ip[i]:ip[i] + pages] != lead:
                    raise ValueError(f"group {g}: sequence {i} does not start with the group's {pages} shared pages")
            s += size

    # -- page-sparse attention ------------------------------------------------------
    def plan_sparse(self, meta: Any, index: Any, budget: int, *, sink: int = 1, recent: int = 1,
                    max_pages: int | None = None) -> SparsePlan:
        """Prepare a step of page-sparse attention: each query and KV head
        attends over at most ``budget`` pages — the first ``sink``, the last
        ``recent`` (its own page included) and the highest scoring others.
        ``max_pages``: a bound on the pages of any sequence of the batch; without
        it the longest is read back from the device once. The plan serves every
        layer of the step; its tables are copies, so ``meta`` may be reused."""
        if index.backend is not self:
            raise ValueError("index belongs to another backend")
        budget, sink, recent = int(budget), int(sink), int(recent)
        if budget <= 0 or sink < 0 or recent < 1 or sink + recent > budget:
            raise ValueError(f"budget={budget}, sink={sink}, recent={recent}: sink >= 0, recent >= 1 and "
                             "sink + recent <= budget are needed")
        plan = SparsePlan()
        self._plan_batch(plan, meta)
        if self.validate == "host":
            self._host_validate(meta, int(meta.query_lens.shape[0]), int(meta.kv_indices.shape[0]))
        if getattr(meta, "batch_indices", None) is None or meta.batch_indices.shape != (plan.n_tokens,):
            raise ValueError(f"plan_sparse needs meta.batch_indices with {plan.n_tokens} entries")
        if max_pages is None:
            ip = plan.tensors["ip"]
            max_pages = int((ip[1:] - ip[:-1]).max())
        if max_pages <= 0:
            raise ValueError(f"max_pages must be positive, got {max_pages}")
        plan.index, plan.budget, plan.sink, plan.recent = index, budget, sink, recent
        plan.max_pages = int(max_pages)
        bi = self._i32(meta.batch_indices)
        rows = plan.tensors["rows"] = torch.empty((plan.n_tokens, 4), dtype=torch.int32, device=self.device)
        plan.rows_ptr = rows.data_ptr()
        N.check(self._lib.pkv_plan_sparse(self._pdesc, plan.batch_ref, bi.data_ptr(), plan.max_pages, plan.rows_ptr,
                                          N.raw_stream(self._dev_index)), "plan_sparse")
        return plan

    def attend_sparse(self, q: torch.Tensor, layer_idx: int, scale: float, plan: SparsePlan, *,
                      out: torch.Tensor | None = None,
                      pages: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Selects each query's pages with the plan's index and attends over
        them, in one launch. Returns ``(out, pages)``: out as ``attend``'s,
        pages int32 ``(tokens, n_kv_heads, budget)`` — page numbers within the
        sequence, ascending, -1 past the end (``pages``: a tensor to write)."""
        return self._sparse(q, layer_idx, scale, plan, out, pages, N.SPARSE_SELECT | N.SPARSE_ATTEND)

    def select_pages(self, q: torch.Tensor, layer_idx: int, plan: SparsePlan, *,
                     pages: torch.Tensor | None = None) -> torch.Tensor:
        """The pages ``attend_sparse`` would read, without the attention."""
        return self._sparse(q, layer_idx, 1.0, plan, None, pages, N.SPARSE_SELECT)[1]

    def attend_pages(self, q: torch.Tensor, layer_idx: int, scale: float, plan: SparsePlan, pages: torch.Tensor, *,
                     out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention over given pages: ``pages`` int32 ``(tokens, n_kv_heads,
        budget)`` as ``select_pages`` returns (another layer's or the caller's
        own). Entries that are negative or past the query's own page are skipped,
        a page listed twice counts twice, a row listing nothing gives zeros."""
        return self._sparse(q, layer_idx, scale, plan, out, pages, N.SPARSE_ATTEND)[0]

    def _sparse(self, q, layer_idx, scale, plan, out, pages, mode):
        if plan.backend is not self:
            raise ValueError("the plan belongs to another backend")
        if layer_idx is None or not 0 <= layer_idx < self.num_layers:
            self._check_layer(layer_idx)
        q = self._query(q, plan.n_tokens)
        if pages is None and mode & N.SPARSE_SELECT:
            pages = torch.empty((plan.n_tokens, self.n_kv_heads, plan.budget), dtype=torch.int32, device=self.device)
        elif (pages is None or pages.shape != (plan.n_tokens, self.n_kv_heads, plan.budget)
              or pages.dtype != torch.int32 or pages.get_device() != self._dev_index or not pages.is_contiguous()):
            raise ValueError(f"pages must be a contiguous int32 {(plan.n_tokens, self.n_kv_heads, plan.budget)} "
                             f"tensor on {self.device}")
        out_ptr = None
        if mode & N.SPARSE_ATTEND:
            out = torch.empty_like(q) if out is None else self._out(q, out)
            out_ptr = out.data_ptr()
        if not plan.n_tokens:
            return out, pages
        rc = self._lib.pkv_attend_sparse(
            self._pdesc, plan.index._pdesc, layer_idx, self.n_heads, q.data_ptr(), out_ptr, pages.data_ptr(), scale,
            plan.budget, plan.sink, plan.recent, plan.batch_ref, plan.rows_ptr, plan.max_pages, mode,
            N.raw_stream(self._dev_index))
        if rc:
            N.check(rc, "attend_sparse")
        if out_ptr:
            self.n_runs += 1
            self.last_kernel = "sparse"
        return out, pages

    def _plan_batch(self, plan: Any, meta: Any) -> None:
        """The step's device tables and batch descriptor of a plan object."""
        plan.backend = self
        n = int(meta.query_lens.shape[0])
        if n <= 0:
            raise ValueError("BatchMeta has no sequences")
        plan.n_tokens = int(meta.positions.shape[0]) if getattr(meta, "positions", None) is not None \
            else int(meta.batch_indices.shape[0])
        t = plan.tensors = {
            "cu": self._copy_i32(meta.cu_query_lens),
            "kl": self._copy_i32(meta.kv_lens) if getattr(meta, "kv_lens", None) is not None else None,
            "ip": self._copy_i32(meta.kv_indptr),
            "ix": self._copy_i32(meta.kv_indices),
            "lp": self._copy_i32(meta.kv_last_page_len),
        }
        total_pages = int(meta.kv_indices.shape[0])
        plan.batch = N.BatchDesc(
            n, plan.n_tokens, total_pages, t["cu"].data_ptr(), N.ptr(t["kl"]), t["ip"].data_ptr(),
            t["ix"].data_ptr() if total_pages else None, t["lp"].data_ptr(), self._status_ptr)
        plan.batch_ref = ctypes.byref(plan.batch)

    def _query(self, q: torch.Tensor, tokens: int) -> torch.Tensor:
        """q checked against the plan's tokens, contiguous in the pool dtype on this device."""
        if q.shape != (tokens, self.n_heads, self.head_dim):
            raise ValueError(f"q has shape {tuple(q.shape)}, expected ({tokens}, {self.n_heads}, {self.head_dim})")
        if q.dtype is self.dtype and q.get_device() == self._dev_index and q.is_contiguous():
            return q
        return q.to(device=self.device, dtype=self.dtype).contiguous()

    def _copy_i32(self, t: torch.Tensor) -> torch.Tensor:
        return t.to(device=self.device, dtype=torch.int32, copy=True).contiguous()

    # -- per-step plan -----------------------------------------------------------

    def plan(self, meta: Any) -> None:
        """Prepare ``meta`` for this step's layers now (validation, device copies
        of the page table, the decode kernel's page schedule). ``attend`` does
        this itself on first sight of a ``meta``; calling it up front keeps that
        work out of the first layer (and inside a captured CUDA graph, if any)."""
        self._step_state(meta)

    def reserve_workspace(self, n_seqs: int, total_pages: int) -> None:
        """Allocate the attention workspace for batches up to this size now, so
        no allocation happens later (e.g. during CUDA-graph capture)."""
        need = int(self._lib.pkv_attend_workspace_size(self._pdesc, self.n_heads, int(n_seqs),
                                                        int(total_pages), 1))
        if self._ws is None or self._ws.numel() < need:
            self._ws = torch.zeros(max(need, 1 << 20), dtype=torch.uint8, device=self.device)
            self.invalidate_plan()

    def _step_state(self, meta: Any) -> dict[str, Any]:
        if self._meta is meta:
            return self._meta_state
        n = int(meta.query_lens.shape[0])
        n_tokens = int(meta.positions.shape[0]) if getattr(meta, "positions", None) is not None \
            else int(meta.batch_indices.shape[0])
        total_pages = int(meta.kv_indices.shape[0])
        if n <= 0:
            raise ValueError("BatchMeta has no sequences")
        # hint for the attention entry point: 1 = every query length is 1 (decode
        # kernel), 2 = none is (pure prefill), 0 = unknown / mixed (the q_len == 1
        # rows of a mixed batch run on the decode kernel)
        checked = int(getattr(meta, "checked_blocks", 0) or 0)
        if self.validate == "host" and not (0 < checked <= self.num_blocks
                                            and getattr(meta, "max_query_len", None) is not None):
            decode, hint = self._host_validate(meta, n, total_pages)
        else:
            # device validation, or an assembler that made the host checks already
            # (DeviceBlockTables: lengths, page counts, block ids inside this pool)
            # is_prefill decides decode vs not (a batch mislabelled as decode is
            # refused below); the query-length bounds only sharpen the hint
            mql = getattr(meta, "max_query_len", None)
            mnql = getattr(meta, "min_query_len", None)
            decode = not bool(meta.is_prefill) if hasattr(meta, "is_prefill") else int(mql) == 1
            hint = 1 if decode else (2 if mnql is not None and int(mnql) > 1 else 0)
        if decode and n_tokens != n:
            raise ValueError(
                f"BatchMeta describes a decode step (is_prefill=False) but has {n_tokens} tokens for "
                f"{n} sequences; a decode step has exactly one query per sequence"
            )
        t = {
            "cu": self._i32(meta.cu_query_lens),
            "kl": self._i32(meta.kv_lens) if getattr(meta, "kv_lens", None) is not None else None,
            "ip": self._i32(meta.kv_indptr),
            "ix": self._i32(meta.kv_indices),
            "lp": self._i32(meta.kv_last_page_len),
        }
        batch = N.BatchDesc(
            n, n_tokens, total_pages, t["cu"].data_ptr(), N.ptr(t["kl"]), t["ip"].data_ptr(),
            t["ix"].data_ptr() if total_pages else None, t["lp"].data_ptr(), self._status.data_ptr(),
        )
        need = int(self._lib.pkv_attend_workspace_size(self._pdesc, self.n_heads, n, total_pages, int(decode)))
        if self._ws is None or self._ws.numel() < need:
            self._ws = torch.zeros(max(need, 1 << 20), dtype=torch.uint8, device=self.device)
        ws_ptr, ws_bytes = self._ws.data_ptr(), self._ws.numel()
        kernel = int(self._lib.pkv_attend_kernel(self._pdesc, self.n_heads, n, n_tokens, hint))
        if kernel < 0:
            N.check(-kernel, "attend")
        if n_tokens > 0 and (decode or kernel == N.PKV_KERNEL_PREFILL):
            N.check(self._lib.pkv_plan(self._pdesc, self.n_heads, ctypes.byref(batch), ws_ptr, ws_bytes,
                                       N.stream_ptr(self.device)), "plan")
            self.n_plans += 1
        self._meta = meta
        self._meta_state = {"batch": batch, "batch_ref": ctypes.byref(batch), "tensors": t, "decode": decode,
                            "hint": hint, "n_tokens": n_tokens,
                            "ws_ptr": ws_ptr, "ws_bytes": ws_bytes, "kernel": N.KERNEL_NAMES[kernel]}
        return self._meta_state

    def _host_validate(self, meta: Any, n: int, total_pages: int) -> tuple[bool, int]:
        """The reference's page-table checks (``paged_torch.py:379-392``) and
        FlashInfer's ``is_prefill`` cross-check (``flashinfer_backend.py:604-618``),
        once per step. Returns (pure decode step, attention hint: 1 all q_len == 1,
        2 none, 0 mixed)."""
        ql = meta.query_lens.tolist()
        ip = meta.kv_indptr.tolist()
        lp = meta.kv_last_page_len.tolist()
        kl = meta.kv_lens.tolist() if getattr(meta, "kv_lens", None) is not None else None
        P = self.block_size
        if len(ip) != n + 1 or ip[0] != 0 or ip[-1] != total_pages:
            raise ValueError(f"kv_indptr must have {n + 1} entries from 0 to {total_pages}")
        for i in range(n):
            pages = ip[i + 1] - ip[i]
            kv_len = kl[i] if kl is not None else (pages - 1) * P + lp[i]
            need = (kv_len + P - 1) // P
            if pages != need:
                raise ValueError(
                    f"{pages} pages supplied but kv_len={kv_len} with block_size={P} needs {need}"
                )
            tail = kv_len - (pages - 1) * P
            if lp[i] != tail:
                raise ValueError(
                    f"kv_last_page_len={lp[i]} but kv_len={kv_len} over {pages} pages implies "
                    f"{tail}. An exact multiple of block_size must report {P}, not 0."
                )
            if ql[i] > kv_len:
                raise ValueError(f"seq {i}: query_len {ql[i]} exceeds kv_len {kv_len}")
        if total_pages:
            ix = meta.kv_indices
            lo, hi = int(ix.min()), int(ix.max())
            if lo < 0 or hi >= self.num_blocks:
                raise ValueError(f"kv_indices outside [0, {self.num_blocks})")
        use_prefill = any(x > 1 for x in ql)
        if hasattr(meta, "is_prefill") and bool(meta.is_prefill) != use_prefill:
            raise ValueError(
                f"BatchMeta.is_prefill={meta.is_prefill} disagrees with query_lens (max={max(ql)}); "
                "is_prefill must be True iff some sequence contributes more than one token"
            )
        if not use_prefill:
            return True, 1
        return False, (0 if any(x == 1 for x in ql) else 2)

    def invalidate_plan(self) -> None:
        """Forget the cached per-step state (for a caller that mutates a
        BatchMeta's tensors in place and reuses the object)."""
        self._meta = None
        self._meta_state = {}
        self._slots_meta = None
        self._slots = None
        self._pos_meta = None
        self._pos = None

    # -- status -----------------------------------------------------------------

    def check_status(self) -> None:
        """Synchronise and raise if any kernel recorded a violation since the
        last check (out-of-pool ids, inconsistent page tables, q_len != 1 in the
        decode kernel, a timed-out device wait)."""
        bits = int(self._status.item())
        if bits:
            self._status.zero_()
            raise N.PkvError(N.PKV_ERR_DEVICE, f"device status {bits:#x}: {N.describe_status(bits)}")

    # -- misc -----------------------------------------------------------------------

    def _i32(self, t: torch.Tensor) -> torch.Tensor:
        return t.to(device=self.device, dtype=torch.int32).contiguous()

    def _out(self, q: torch.Tensor, out: torch.Tensor | None) -> torch.Tensor:
        if out is None:
            return torch.empty_like(q)
        if (out.shape != q.shape or out.dtype != self.dtype or not out.is_cuda
                or out.get_device() != self._dev_index or not out.is_contiguous()):
            raise ValueError(f"out must be a contiguous {tuple(q.shape)} {self.dtype} tensor on {self.device}")
        nb = q.numel() * q.element_size()
        if out.data_ptr() < q.data_ptr() + nb and q.data_ptr() < out.data_ptr() + nb:
            raise ValueError("out must not overlap q (other CTAs may still read a row being written)")
        return out

    def _own(self, t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
        """t on this device in `dtype`, contiguous (no op when it already is)."""
        if t.is_cuda and t.dtype == dtype and t.get_device() == self._dev_index and t.is_contiguous():
            return t
        return t.to(device=self.device, dtype=dtype).contiguous()

    def _check_layer(self, layer_idx: int) -> None:
        if layer_idx is None or not 0 <= layer_idx < self.num_layers:
            raise ValueError(f"layer_idx {layer_idx} out of range [0, {self.num_layers})")

    def reset(self) -> None:
        """Zero every pool and its indexes and drop the cached step state. Tests only."""
        self._pool.zero_()
        for ref in self._indexes:
            if (index := ref()) is not None:
                index.codes.zero_()
                index.scales.zero_()
        self.invalidate_plan()

    def __repr__(self) -> str:
        mib = self.pool_bytes() / (1024 * 1024)
        return (
            f"B200PagedBackend(layers={self.num_layers}, blocks={self.num_blocks}, "
            f"block_size={self.block_size}, kv_heads={self.n_kv_heads}, heads={self.n_heads}, "
            f"head_dim={self.head_dim}, dtype={self.dtype}, device={self.device}, pool={mib:.1f} MiB)"
        )


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the address ranges of two tensors meet."""
    def span(t):
        n = 1 + sum((d - 1) * st for d, st in zip(t.shape, t.stride())) if t.numel() else 0
        return t.data_ptr(), t.data_ptr() + n * t.element_size()

    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1

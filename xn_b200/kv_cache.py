"""A KV cache held in GGUF blocks (Q4_0 or Q8_0 along ``head_dim``): written as tokens arrive, read back, attended to.

The cache of a Llama-style decoder in bf16 takes 512 bytes a position and KV head of 128 (keys and values), and a decode step reads all of it; as Q4_0
blocks it is 144 bytes, as Q8_0 272. ``QLlama(kv_dtype=...)`` uses it; any other program can::

    cache = QuantizedKVCache(GgmlDType.Q4_0, batch, kv_heads, max_seq, head_dim, device)
    cache.store(k, v, pos)                                # k, v [batch, seq, kv_heads, head_dim]; pos [batch] int64 on the device
    q = cache.rope_store(qkv, cos, sin, pos, heads)       # or: the fused projection's output, rotary embedding included
    out = cache.attend(q, pos)                            # q [batch, seq, heads, head_dim]: one token, a few drafts, a prompt
    k, v = cache.load(0, n)                               # what the blocks stand for

Between requests, all of it on the GPU and without a look at the results::

    room, free = cache.reserve(length)                    # the page table brought to the requests' lengths
    plan = cache.plan(pos, count, tokens)                 # sequences of their own numbers of tokens, packed one after the other
    q = cache.rope_store(qkv, cos, sin, plan, heads)      # the calls above with a plan for pos; qkv [tokens, ..], q [tokens, heads, head_dim]
    out = cache.attend(q, plan, window=4096, sinks=4)     # a window, and first positions that stay visible
    plan = cache.plan(pos, count, tokens, longest, parents)   # trees of drafted tokens: each sees its ancestors
    pos = cache.keep(plan, node)                          # the accepted path stays

``pos`` is the position of the first of a call's ``seq`` tokens, one for every sequence or one for all. A token at a negative position is none (an idle slot of
the batch, padding on the left): it is not stored, and its query gives zeros. Everything is enqueued on the current stream. There are no derivatives: tensors
that require a gradient are refused, but under ``torch.no_grad()``, and so are tracers.
"""
from __future__ import annotations

import contextlib
import ctypes
import threading
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from .dtypes import GgmlDType
from .quantized import _TORCH_TO_XNQ, _XNQ_IDS, _stream_ptr, init

TREE_MOST = 256  # tokens of a tree: XNQ_KV_TREE_MOST
_ZEROED = 4096  # XNQ_KV_WORKSPACE_ZEROED: the front of attention's workspace, zero before its first use
PAGE_UNIT = 32  # positions of a tile: page sizes are multiples of it


class _Cache(ctypes.Structure):
    _fields_ = [("ggml_dtype", ctypes.c_int), ("kv_heads", ctypes.c_int), ("head_dim", ctypes.c_int), ("page_size", ctypes.c_int64), ("num_pages", ctypes.c_int64),
                ("pages", ctypes.c_void_p), ("page_table", ctypes.c_void_p), ("table_stride", ctypes.c_int64), ("max_seq", ctypes.c_int64)]


class _Rows(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("dtype", ctypes.c_int), ("stride_b", ctypes.c_int64), ("stride_s", ctypes.c_int64), ("stride_h", ctypes.c_int64)]


class _Rope(ctypes.Structure):
    _fields_ = [("cos_table", ctypes.c_void_p), ("sin_table", ctypes.c_void_p), ("table_rows", ctypes.c_int64), ("heads", ctypes.c_int), ("q", _Rows), ("q_out", _Rows)]


class _Plan(ctypes.Structure):
    _fields_ = [("tokens", ctypes.c_int64), ("batch", ctypes.c_int64), ("longest", ctypes.c_int64), ("start", ctypes.c_void_p), ("offsets", ctypes.c_void_p),
                ("sequence", ctypes.c_void_p), ("position", ctypes.c_void_p), ("slot", ctypes.c_void_p), ("sees", ctypes.c_void_p), ("nodes", ctypes.c_void_p)]


def _served(t: torch.Tensor) -> bool:
    """Whether the kernels can read this [batch, seq, heads, head_dim] or [tokens, heads, head_dim] tensor where it lies: rows contiguous and 16-byte aligned."""
    e = 16 // t.element_size()
    return t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s % e == 0 for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1)


def _rows(t: torch.Tensor) -> _Rows:
    strides = [s if n > 1 else 0 for s, n in zip(t.stride()[:-1], t.shape[:-1])]   # of a dimension of one entry torch may say anything
    return _Rows(t.data_ptr(), int(_TORCH_TO_XNQ[t.dtype]), *([0] * (3 - len(strides))), *strides)


def _refuse_derivatives(who: str, *tensors: Optional[torch.Tensor]) -> None:
    """These calls are torch operators of no kind: no gradient, tangent or trace comes out of them, and a call that asks for one says so."""
    if torch._C._get_tracing_state() is not None:
        raise RuntimeError(f"{who} cannot be traced")
    for t in tensors:
        if isinstance(t, torch.Tensor) and ((t.requires_grad and torch.is_grad_enabled()) or (forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None)):
            raise RuntimeError(f"{who} has no derivative, and one of its tensors asks for it: call it under torch.no_grad(), or with detached tensors")


_MOST_WORKSPACES = 16   # streams that have scratch of their own; a call of another one takes and clears its own
_workspaces: dict[tuple[int, int], tuple[torch.Tensor, threading.Lock]] = {}   # (device, stream) -> zeroed once; a kernel leaves its counters at zero
_NO_LOCK = contextlib.nullcontext()


def _workspace(device: torch.device, need: int):
    """Scratch on the current stream, and the lock to hold while a call that uses it is enqueued (its kernels follow one another on the stream)."""
    capturing = torch.cuda.is_current_stream_capturing()   # a graph may be replayed beside others: scratch of its own, zeroed in every replay
    key = (device.index, int(_stream_ptr(device).value or 0))
    kept = None if capturing else _workspaces.get(key)
    if kept is not None and kept[0].numel() >= need:
        return kept
    if capturing or (kept is None and len(_workspaces) >= _MOST_WORKSPACES):
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        ws[:_ZEROED].zero_()
        return ws, _NO_LOCK
    kept = _workspaces[key] = (torch.zeros(need, dtype=torch.uint8, device=device), threading.Lock())
    return kept


class KVPlan:
    """Where the tokens of a step go: made by :meth:`QuantizedKVCache.plan`, good for every cache with the same page table (a model's layers).

    ``offsets`` int64 ``[batch + 1]``: sequence ``b`` has the rows ``offsets[b] ..`` of the packed tokens. ``sequence`` (int32), ``position`` and ``slot`` (int64)
    ``[tokens]``: of each row its sequence, the position that it is rotated at, and ``page * page_size + place`` in the cache's memory; -1: none. ``start``:
    ``pos``, as it was. For trees ``sees`` (int32 ``[tokens, ceil(longest / 32)]``, bit ``t % 32`` of word ``t // 32``: the token sees token ``t`` of its tree) and
    ``nodes`` (the same for all tokens of a tree ``[batch, ..]``); else None. The tensors are the plan's own and not to be written to."""

    __slots__ = ("tokens", "longest", "batch", "start", "offsets", "sequence", "position", "slot", "sees", "nodes", "_handle")

    def __init__(self, tokens: int, longest: int, batch: int, made: tuple):
        self.tokens, self.longest, self.batch = tokens, longest, batch
        self._handle, self.start, self.offsets, self.sequence, self.position, self.slot, self.sees, self.nodes = made


class QuantizedKVCache:
    """Keys and values of ``batch`` sequences of up to ``max_seq`` positions, ``dtype`` blocks (Q4_0, Q8_0), ``head_dim`` 64 or 128.

    ``page_size`` (a multiple of 32): the memory is ``num_pages`` pages of that many positions, and ``page_table`` (int32 ``[batch, ceil(max_seq /
    page_size)]`` on the device, all -1 at first) says which page holds positions ``i * page_size ..`` of a sequence; :meth:`reserve` or the program fills it in
    (in place: the kernels hold its address, and a cache's attributes are not exchanged). ``page_table``: another cache's, which this one shares (the layers
    of a model: one :meth:`reserve` for all). Without pages every sequence has one run of memory."""

    _FIXED = frozenset(("pages", "page_table", "dtype", "batch", "kv_heads", "max_seq", "head_dim", "page_size", "num_pages", "device"))

    def __setattr__(self, name, value):
        if name in self._FIXED and name in self.__dict__:
            raise AttributeError(f"QuantizedKVCache.{name} is fixed when the cache is made" + (": fill it in place" if name in ("pages", "page_table") else ""))
        super().__setattr__(name, value)

    def __init__(self, dtype: GgmlDType, batch: int, kv_heads: int, max_seq: int, head_dim: int, device: torch.device | str = "cuda:0",
                 page_size: Optional[int] = None, num_pages: Optional[int] = None, page_table: Optional[torch.Tensor] = None):
        self.dtype, self.batch, self.kv_heads, self.max_seq, self.head_dim = GgmlDType(dtype), batch, kv_heads, max_seq, head_dim
        if min(batch, kv_heads, max_seq) < 1:
            raise ValueError(f"QuantizedKVCache: batch {batch}, kv_heads {kv_heads}, max_seq {max_seq}")
        if (page_size is None) != (num_pages is None):
            raise ValueError("QuantizedKVCache: page_size and num_pages go together")
        paged = page_size is not None
        self.page_size = page_size if paged else -(-max_seq // PAGE_UNIT) * PAGE_UNIT
        self.num_pages = num_pages if paged else batch
        page_bytes = int(_lib.lib().xnq_kv_page_bytes(int(self.dtype), kv_heads, head_dim, self.page_size))
        if page_bytes == 0 or self.num_pages < 1:
            raise ValueError(f"QuantizedKVCache: no cache of {self.dtype.name} blocks, {kv_heads} heads of {head_dim}, {self.num_pages} pages of {self.page_size} "
                             f"positions (Q4_0 or Q8_0; heads of 64 or 128; pages of a multiple of {PAGE_UNIT})")
        device = torch.device(device)
        self.device = torch.device("cuda", torch.cuda.current_device()) if device.index is None else device
        init(self.device)
        self.pages = torch.zeros((self.num_pages, page_bytes), dtype=torch.uint8, device=self.device)
        shape = (batch, -(-max_seq // self.page_size))
        if page_table is not None and (not paged or page_table.shape != shape or page_table.dtype is not torch.int32 or page_table.device != self.device or not page_table.is_contiguous()):
            raise ValueError(f"QuantizedKVCache: page_table is contiguous int32 {shape} on {self.device}, of a cache by pages")
        self.page_table = page_table if page_table is not None else torch.full(shape, -1, dtype=torch.int32, device=self.device) if paged else None
        self._view = _Cache(int(self.dtype), kv_heads, head_dim, self.page_size, self.num_pages, self.pages.data_ptr(),
                            self.page_table.data_ptr() if paged else None, shape[1] if paged else 0, max_seq)

        self._native = _lib.native()   # the ordinary call, in C++ (csrc/torch_kv_cache.cpp); what it hands back as None is taken here
        self._handle = self._native.kv_cache(ctypes.addressof(self._view), batch, self.device.index)

    @property
    def nbytes(self) -> int:
        return self.pages.numel()

    def _tokens(self, what: str, t: torch.Tensor, heads: Optional[int] = None) -> torch.Tensor:
        if t.dim() != 4 or t.shape[0] != self.batch or t.shape[3] != self.head_dim or (heads is not None and t.shape[2] != heads):
            raise ValueError(f"{what} is {tuple(t.shape)}; the cache holds {self.batch} sequences, {self.kv_heads} KV heads of {self.head_dim}")
        if t.device != self.device:
            raise ValueError(f"{what} is on {t.device}, the cache on {self.device}")
        if t.dtype not in _TORCH_TO_XNQ:
            raise ValueError(f"{what} is {t.dtype}; float32, float16 and bfloat16 are served")
        return t

    def _positions(self, pos: torch.Tensor, what: str = "pos"):
        """Its address and stride (0: one position for all)."""
        if pos.dtype is not torch.int64 or pos.device != self.device or not pos.is_contiguous() or pos.numel() not in (1, self.batch):
            raise ValueError(f"{what}: int64 on {self.device}, one for each of the {self.batch} sequences or one for all")
        return ctypes.c_void_p(pos.data_ptr()), int(pos.numel() > 1)

    def reserve(self, length: torch.Tensor, first: Optional[torch.Tensor] = None, sinks: int = 0, table: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Bring the page table to the requests' lengths: sequence ``b`` has a page wherever positions below ``length[b]`` (int64 ``[batch]``; 0: no request)
        need one, and none beyond. Pages that are there stay; the others come, in ascending order, from those that no row names any more (a page that two rows
        name, a shared beginning, is free when both have let go). ``first`` (int64 ``[batch]``): positions below it are seen no more, but for the first
        ``sinks``, and their pages are given back (attention with a window). ``table``: what to start from, instead of the table as it is (its shape and type).

        Returns ``room`` int64 ``[batch]``, the positions that there are pages for (``length``, or less where the pages did not suffice: sequences in their
        order, each up to its first missing page), and ``free`` int64 ``[]``, the pages left."""
        if self.page_table is None:
            raise ValueError("reserve: this cache has no pages")
        both = self._native.kv_reserve(self._handle, self.page_table, self.page_table if table is None else table, length, first, sinks)
        if both is not None:
            return both
        _refuse_derivatives("reserve")
        for what, t in (("length", length), ("first", first)):
            if t is not None and (t.dtype is not torch.int64 or t.device != self.device or t.shape != (self.batch,) or not t.is_contiguous()):
                raise ValueError(f"reserve: {what} is contiguous int64 [{self.batch}] on {self.device}")
        if sinks < 0:
            raise ValueError(f"reserve: sinks {sinks}")
        if table is None:
            table = self.page_table
        elif table.shape != self.page_table.shape or table.dtype is not torch.int32 or table.device != self.device or not table.is_contiguous():
            raise ValueError(f"reserve: table is contiguous int32 {tuple(self.page_table.shape)} on {self.device}")
        out = torch.empty(self.batch + 1, dtype=torch.int64, device=self.device)
        L = _lib.lib()
        need = int(L.xnq_kv_reserve_workspace_bytes(self.batch, self.page_size, self.num_pages, self.max_seq))
        with torch.cuda.device(self.device):
            ws = torch.empty(max(need, 16), dtype=torch.uint8, device=self.device)
            p = lambda t: None if t is None else ctypes.c_void_p(t.data_ptr())
            _lib.check(L.xnq_kv_reserve(p(self.page_table), table.shape[1], p(table), table.shape[1], self.batch, self.page_size, self.num_pages, self.max_seq,
                                        p(length), p(first), sinks, p(out), ctypes.c_void_p(out.data_ptr() + 8 * self.batch), p(ws), need, _stream_ptr(self.device)))
        return out[:-1], out[-1]

    def plan(self, pos: torch.Tensor, count: torch.Tensor, tokens: int, longest: Optional[int] = None, parents: Optional[torch.Tensor] = None) -> KVPlan:
        """Slot maps of packed tokens: sequence ``b`` brings ``count[b]`` (int64 ``[batch]``) tokens for the positions ``pos[b] ..``, all of them lie one after
        the other in ``tokens`` rows; rows behind the last sequence are none. ``longest``: no sequence brings more (default ``tokens``). What is beyond
        ``longest`` or ``tokens`` is cut off, and sets a status bit.

        ``parents`` (int32 ``[tokens]``): the tokens of a sequence are a tree of drafts. Each one's is the index, in its sequence, of the token that it follows (a
        smaller one than its own); -1: it follows what is in the cache; -2: the place is not used. They lie at ``pos, pos + 1, ..`` in the cache, in their
        order, are rotated at ``pos`` + depth, and see what lies below ``pos`` and their ancestors. Up to 256 tokens a tree.

        The plan holds the slots of the page table as it is when the call runs: after :meth:`reserve`, before the calls that take it. It is made on the current
        stream; another stream that takes it waits for this one first, or reads what is not there yet."""
        if tokens < 0 or (longest is not None and longest < 1):
            raise ValueError(f"plan: {tokens} tokens, up to {longest} a sequence")
        longest = max(1, min(tokens, longest if longest is not None else tokens))
        made = self._native.kv_plan(self._handle, pos, count, tokens, longest, parents)
        if made is not None:
            return KVPlan(tokens, longest, self.batch, made)
        _refuse_derivatives("plan")
        if count.dtype is not torch.int64 or count.device != self.device or count.shape != (self.batch,) or not count.is_contiguous():
            raise ValueError(f"plan: count is contiguous int64 [{self.batch}] on {self.device}")
        if parents is not None:
            if parents.dtype is not torch.int32 or parents.device != self.device or parents.shape != (tokens,) or not parents.is_contiguous():
                raise ValueError(f"plan: parents is contiguous int32 [{tokens}] on {self.device}")
            if longest > TREE_MOST:
                raise ValueError(f"plan: trees of up to {longest} tokens (up to {TREE_MOST} are served)")
        pp, stride = self._positions(pos)
        b, words = self.batch, -(-longest // 32) if parents is not None else 0
        with torch.cuda.device(self.device):
            wide = torch.empty(2 * b + 1 + 2 * tokens + 1, dtype=torch.int64, device=self.device)   # (one more than there are: no address is null)
            narrow = torch.empty(tokens + (tokens + b) * words + 1, dtype=torch.int32, device=self.device)
            start, offsets, position, slot, _ = wide.split([b, b + 1, tokens, tokens, 1])
            sequence, sees, nodes, _ = narrow.split([tokens, tokens * words, b * words, 1])
            w, n = wide.data_ptr(), narrow.data_ptr()
            tree = parents is not None
            view = _Plan(tokens, b, longest, w, w + 8 * b, n, w + 8 * (2 * b + 1), w + 8 * (2 * b + 1 + tokens), n + 4 * tokens if tree else None, n + 4 * (tokens + tokens * words) if tree else None)
            _lib.check(_lib.lib().xnq_kv_plan_make(ctypes.byref(self._view), pp, stride, ctypes.c_void_p(count.data_ptr()),
                                                   ctypes.c_void_p(parents.data_ptr() or n) if tree else None, ctypes.byref(view), _stream_ptr(self.device)))
        table = self.page_table.data_ptr() if self.page_table is not None else 0
        handle = self._native.kv_plan_handle(ctypes.addressof(view), table, self.page_size, self.num_pages, self.max_seq, self.device.index)
        return KVPlan(tokens, longest, b, (handle, start, offsets, sequence, position, slot, sees.view(tokens, words) if tree else None, nodes.view(b, words) if tree else None))

    def _planned(self, who: str, plan: KVPlan) -> ctypes.c_void_p:
        """The address of the plan's description. Its slots have to be this cache's."""
        view, *made_for = self._native.kv_plan_view(plan._handle)
        if plan.batch != self.batch or made_for != [self.page_table.data_ptr() if self.page_table is not None else 0, self.page_size, self.num_pages, self.max_seq, self.device.index]:
            raise ValueError(f"{who}: the plan was made for another cache (its device, batch, pages and page table have to be this one's)")
        return ctypes.c_void_p(view)

    def keep(self, plan: KVPlan, node: torch.Tensor) -> torch.Tensor:
        """Of each tree of drafted tokens the path to ``node[b]`` (int64 ``[batch]``, the index in its tree; -1: no token) stays: the keys and values of its
        tokens move up to the positions ``pos[b], pos[b] + 1, ..``. Returns where each sequence goes on, int64 ``[batch]``: ``pos`` plus the path's length. What
        the other tokens had stored may lie behind that."""
        if isinstance(plan, KVPlan):
            pos = self._native.kv_keep(self._handle, plan._handle, node)
            if pos is not None:
                return pos
        _refuse_derivatives("keep")
        view = self._planned("keep", plan)
        if plan.sees is None:
            raise ValueError("keep: the plan is not one of trees (parents)")
        if node.dtype is not torch.int64 or node.device != self.device or node.shape != (self.batch,) or not node.is_contiguous():
            raise ValueError(f"keep: node is contiguous int64 [{self.batch}] on {self.device}")
        with torch.cuda.device(self.device):
            pos = torch.empty(self.batch, dtype=torch.int64, device=self.device)
            _lib.check(_lib.lib().xnq_kv_keep(ctypes.byref(self._view), view, ctypes.c_void_p(node.data_ptr()), ctypes.c_void_p(pos.data_ptr()),
                                              _stream_ptr(self.device)))
        return pos

    def _packed(self, what: str, t: torch.Tensor, plan: KVPlan, heads: Optional[int] = None) -> torch.Tensor:
        if t.dim() != 3 or t.shape[0] != plan.tokens or t.shape[2] != self.head_dim or (heads is not None and t.shape[1] != heads):
            raise ValueError(f"{what} is {tuple(t.shape)}; the plan has {plan.tokens} tokens, the cache {self.kv_heads} KV heads of {self.head_dim}")
        if t.device != self.device:
            raise ValueError(f"{what} is on {t.device}, the cache on {self.device}")
        if t.dtype not in _TORCH_TO_XNQ:
            raise ValueError(f"{what} is {t.dtype}; float32, float16 and bfloat16 are served")
        return t

    def store(self, k: torch.Tensor, v: torch.Tensor, pos: torch.Tensor | KVPlan) -> None:
        """Quantize ``k`` and ``v`` ``[batch, seq, kv_heads, head_dim]`` (f32 / f16 / bf16, any strides) into positions ``pos ..``: the blocks that
        ``BlockQ4_0`` / ``BlockQ8_0::from_float`` make of the f32 values (k_quants.rs:235-270, 636-661), Q8_0's scale being ``max|x| * float32(1 / 127)``.
        With a plan: ``[tokens, kv_heads, head_dim]``, each token into its slot."""
        plan = pos if isinstance(pos, KVPlan) else None
        if self._native.kv_store(self._handle, k, v, pos if plan is None else plan._handle):
            return
        if plan is not None:
            _refuse_derivatives("store", k, v)
            view = self._planned("store", plan)
            self._packed("k", k, plan, self.kv_heads), self._packed("v", v, plan, self.kv_heads)
            if k.dtype is not v.dtype:
                raise ValueError(f"k is {k.dtype}, v {v.dtype}")
            return self._store_packed(k, v, plan.tokens, view, None)
        _refuse_derivatives("store", k, v)
        self._tokens("k", k, self.kv_heads), self._tokens("v", v, self.kv_heads)
        if k.shape != v.shape or k.dtype is not v.dtype:
            raise ValueError(f"k is {tuple(k.shape)} {k.dtype}, v {tuple(v.shape)} {v.dtype}")
        self._store(k, v, pos, None)

    def rope_store(self, qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, pos: torch.Tensor | KVPlan, heads: int, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """``qkv`` ``[batch, seq, (heads + 2 kv_heads) * head_dim]``, a fused projection's output: q and k rotated (rotate-half, f32 tables ``[rows, head_dim /
        2]``) at their positions, k and v stored. Returns q ``[batch, seq, heads, head_dim]`` as ``out_dtype`` (default: ``qkv``'s). With a plan: ``[tokens, ..]``,
        and q ``[tokens, heads, head_dim]``, zeros for rows that are no token."""
        plan = pos if isinstance(pos, KVPlan) else None
        if out_dtype is None or out_dtype in _TORCH_TO_XNQ:
            q = self._native.kv_rope_store(self._handle, qkv, cos, sin, pos if plan is None else plan._handle, heads, -1 if out_dtype is None else _XNQ_IDS[out_dtype])
            if q is not None:
                return q
        _refuse_derivatives("rope_store", qkv, cos, sin)
        hd, width = self.head_dim, (heads + 2 * self.kv_heads) * self.head_dim
        view = None if plan is None else self._planned("rope_store", plan)
        if heads < 1 or qkv.dim() != (3 if plan is None else 2) or qkv.shape[-1] != width:
            raise ValueError(f"rope_store: qkv is {tuple(qkv.shape)}; {heads} + 2 * {self.kv_heads} heads of {hd}")
        for t in (cos, sin):
            if t.dtype is not torch.float32 or not t.is_contiguous() or t.dim() != 2 or t.shape[1] != hd // 2 or t.shape != cos.shape or t.device != self.device:
                raise ValueError(f"rope_store: tables are contiguous float32 [rows, {hd // 2}] on {self.device}")
        if out_dtype is not None and out_dtype not in _TORCH_TO_XNQ:
            raise ValueError(f"rope_store: queries of type {out_dtype}")
        x = qkv.unflatten(-1, (-1, hd))
        if not _served(x):
            x = x.clone(memory_format=torch.contiguous_format)
        self._tokens("qkv", x) if plan is None else self._packed("qkv", x, plan)
        q, k, v = x.split([heads, self.kv_heads, self.kv_heads], dim=-2)
        out = torch.empty((*q.shape,), dtype=out_dtype or qkv.dtype, device=self.device)
        if out.numel():
            rope = _Rope(cos.data_ptr(), sin.data_ptr(), cos.shape[0], heads, _rows(q), _rows(out))
            self._store(k, v, pos, rope) if plan is None else self._store_packed(k, v, plan.tokens, view, rope)
        return out

    def _store_packed(self, k, v, tokens, view, rope) -> None:
        if tokens == 0:
            return
        k, v = (t if _served(t) else t.clone(memory_format=torch.contiguous_format) for t in (k, v))
        with torch.cuda.device(self.device):
            _lib.check(_lib.lib().xnq_kv_store_packed(ctypes.byref(self._view), ctypes.byref(_rows(k)), ctypes.byref(_rows(v)), view,
                                                      None if rope is None else ctypes.byref(rope), _stream_ptr(self.device)))

    def _store(self, k, v, pos, rope) -> None:
        k, v = (t if _served(t) else t.clone(memory_format=torch.contiguous_format) for t in (k, v))
        pp, stride = self._positions(pos)
        with torch.cuda.device(self.device):
            _lib.check(_lib.lib().xnq_kv_store(ctypes.byref(self._view), ctypes.byref(_rows(k)), ctypes.byref(_rows(v)), self.batch, k.shape[1], pp, stride,
                                               None if rope is None else ctypes.byref(rope), _stream_ptr(self.device)))

    def load(self, start: int | torch.Tensor, length: int, dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values ``[batch, kv_heads, length, head_dim]`` of positions ``start ..`` (a number, or int64 on the device as ``pos``), as ``dtype``: scale
        times code, in f32, rounded once. Positions that are not in the cache or have no page are zeros."""
        if dtype not in _TORCH_TO_XNQ or length < 0:
            raise ValueError(f"load: {length} positions as {dtype}")
        both = self._native.kv_load(self._handle, start, length, _XNQ_IDS[dtype])
        if both is not None:
            return both
        _refuse_derivatives("load")
        k = torch.empty((self.batch, self.kv_heads, length, self.head_dim), dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        sp, stride = self._positions(start, "start") if isinstance(start, torch.Tensor) else (None, 0)
        with torch.cuda.device(self.device):
            _lib.check(_lib.lib().xnq_kv_load(ctypes.byref(self._view), self.batch, sp, stride, 0 if sp else int(start), length, int(_TORCH_TO_XNQ[dtype]),
                                              ctypes.c_void_p(k.data_ptr()), ctypes.c_void_p(v.data_ptr()), _stream_ptr(self.device)))
        return k, v

    def attend(self, q: torch.Tensor, pos: torch.Tensor | KVPlan, causal: bool = True, window: int = 0, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
               lse: Optional[torch.Tensor] = None, sinks: int = 0) -> torch.Tensor:
        """Attention of ``q`` ``[batch, seq, heads, head_dim]`` (f32 / f16 / bf16, any strides) over the cache; ``heads`` is a multiple of ``kv_heads``.

        Query ``i`` of a sequence is at ``p = pos + i`` and sees positions ``j <= p`` (``causal``) or ``j < pos + seq``, with a ``window`` only ``j > p - window``
        and, of the others, the first ``sinks``; one that sees nothing gives zeros. ``scale``: default ``head_dim ** -0.5``. ``out``: where the result goes
        (``q``'s shape and type, rows contiguous and 16-byte aligned). ``lse``: float32 ``[batch, seq, heads]`` that receives the logarithm of the sum of
        exponentials (-inf: nothing seen).

        With a plan: ``q`` ``[tokens, heads, head_dim]``, ``lse`` ``[tokens, heads]``. A token of a tree sees what lies below its tree, with a ``window`` (at
        least ``plan.longest``) as one at ``p`` = its position does, and its ancestors in the tree, whatever ``causal``. Rows that are no token give zeros; those
        behind the last sequence are left as they are where ``out`` is given.

        Many 16-bit rows with a ``window`` take less time with a plan or ``sinks`` than without either (2048 tokens, a window of 4096: 189 us against 335)."""
        plan = pos if isinstance(pos, KVPlan) else None
        if out is None and lse is None:
            res = self._native.kv_attend(self._handle, q, pos if plan is None else plan._handle, causal, window, self.head_dim ** -0.5 if scale is None else scale, sinks)
            if res is not None:
                return res
        _refuse_derivatives("attend", q, out, lse)
        view = None
        if plan is not None:
            view = self._planned("attend", plan)
            self._packed("q", q, plan)
        else:
            self._tokens("q", q)
        heads = q.shape[-2]
        batch, seq = (self.batch, q.shape[1]) if plan is None else (plan.batch, plan.longest)
        if heads < 1 or heads % self.kv_heads:
            raise ValueError(f"attend: {heads} query heads over {self.kv_heads} KV heads")
        if window < 0 or sinks < 0:
            raise ValueError(f"attend: window {window}, sinks {sinks}")
        if plan is not None and plan.sees is not None and 0 < window < plan.longest:
            raise ValueError(f"attend: a window of {window} is shorter than the plan's trees of up to {plan.longest} tokens")
        clear = out is None
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=self.device)
        elif out.shape != q.shape or out.dtype is not q.dtype or out.device != self.device or not _served(out) or any(s == 0 and n > 1 for s, n in zip(out.stride(), out.shape)):
            raise ValueError(f"attend: out is {tuple(out.shape)} {out.dtype}; q is {tuple(q.shape)} {q.dtype}, and rows are contiguous, apart and 16-byte aligned")
        if lse is not None and (lse.shape != q.shape[:-1] or lse.dtype is not torch.float32 or lse.device != self.device or not lse.is_contiguous()):
            raise ValueError(f"attend: lse is contiguous float32 {tuple(q.shape[:-1])}")
        if not _served(q):
            q = q.clone(memory_format=torch.contiguous_format)
        pp, stride = self._positions(pos) if plan is None else (None, 0)
        if out.numel() == 0:
            return out
        L = _lib.lib()
        common = (self.head_dim ** -0.5 if scale is None else float(scale), int(causal), int(window))
        rows = (ctypes.byref(self._view), ctypes.byref(_rows(q)), ctypes.byref(_rows(out)), None if lse is None else ctypes.c_void_p(lse.data_ptr()))
        with torch.cuda.device(self.device):
            need = L.xnq_kv_attend_workspace_bytes(batch, seq, heads, self.kv_heads, self.head_dim) if plan is None else \
                L.xnq_kv_attend_packed_workspace_bytes(view, heads, self.kv_heads, self.head_dim)
            ws, lock = _workspace(self.device, max(16, int(need)))
            scratch = (ctypes.c_void_p(ws.data_ptr()), ws.numel(), _stream_ptr(self.device))
            with lock:   # (the interpreter's is free during the call, which may enqueue two kernels)
                if plan is None and not (sinks and window):
                    rc = L.xnq_kv_attend(*rows, batch, seq, heads, pp, stride, *common, *scratch)
                else:
                    rc = L.xnq_kv_attend_packed(*rows, batch, seq, heads, pp, stride, view, int(clear), *common, int(sinks), *scratch)
            _lib.check(rc)
        return out

"""A KV cache held in GGUF blocks (Q4_0 or Q8_0 along ``head_dim``): written as tokens arrive, read back, attended to.

The cache of a Llama-style decoder in bf16 takes 512 bytes a position and KV head of 128 (keys and values), and a decode step reads all of it; as Q4_0
blocks it is 144 bytes, as Q8_0 272. ``QLlama(kv_dtype=...)`` uses it; any other program can::

    cache = QuantizedKVCache(GgmlDType.Q4_0, batch, kv_heads, max_seq, head_dim, device)
    cache.store(k, v, pos)                                # k, v [batch, seq, kv_heads, head_dim]; pos [batch] int64 on the device
    q = cache.rope_store(qkv, cos, sin, pos, heads)       # or: the fused projection's output, rotary embedding included
    out = cache.attend(q, pos)                            # q [batch, seq, heads, head_dim]: one token, a few drafts, a prompt
    k, v = cache.load(0, n)                               # what the blocks stand for

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

_ZEROED = 4096  # XNQ_KV_WORKSPACE_ZEROED: the front of attention's workspace, zero before its first use
PAGE_UNIT = 32  # positions of a tile: page sizes are multiples of it


class _Cache(ctypes.Structure):
    _fields_ = [("ggml_dtype", ctypes.c_int), ("kv_heads", ctypes.c_int), ("head_dim", ctypes.c_int), ("page_size", ctypes.c_int64), ("num_pages", ctypes.c_int64),
                ("pages", ctypes.c_void_p), ("page_table", ctypes.c_void_p), ("table_stride", ctypes.c_int64), ("max_seq", ctypes.c_int64)]


class _Rows(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("dtype", ctypes.c_int), ("stride_b", ctypes.c_int64), ("stride_s", ctypes.c_int64), ("stride_h", ctypes.c_int64)]


class _Rope(ctypes.Structure):
    _fields_ = [("cos_table", ctypes.c_void_p), ("sin_table", ctypes.c_void_p), ("table_rows", ctypes.c_int64), ("heads", ctypes.c_int), ("q", _Rows), ("q_out", _Rows)]


def _served(t: torch.Tensor) -> bool:
    """Whether the kernels can read this [batch, seq, heads, head_dim] tensor where it lies: rows contiguous and 16-byte aligned."""
    e = 16 // t.element_size()
    return t.stride(3) == 1 and t.data_ptr() % 16 == 0 and all(s % e == 0 for s, n in zip(t.stride()[:3], t.shape[:3]) if n > 1)


def _rows(t: torch.Tensor) -> _Rows:
    strides = [s if n > 1 else 0 for s, n in zip(t.stride()[:3], t.shape[:3])]   # of a dimension of one entry torch may say anything
    return _Rows(t.data_ptr(), int(_TORCH_TO_XNQ[t.dtype]), *strides)


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


class QuantizedKVCache:
    """Keys and values of ``batch`` sequences of up to ``max_seq`` positions, ``dtype`` blocks (Q4_0, Q8_0), ``head_dim`` 64 or 128.

    ``page_size`` (a multiple of 32): the memory is ``num_pages`` pages of that many positions, and ``page_table`` (int32 ``[batch, ceil(max_seq /
    page_size)]`` on the device, all -1 at first) says which page holds positions ``i * page_size ..`` of a sequence; the program fills it in (in place: the
    kernels hold its address, and a cache's attributes are not exchanged). Without it every sequence has one run of memory."""

    _FIXED = frozenset(("pages", "page_table", "dtype", "batch", "kv_heads", "max_seq", "head_dim", "page_size", "num_pages", "device"))

    def __setattr__(self, name, value):
        if name in self._FIXED and name in self.__dict__:
            raise AttributeError(f"QuantizedKVCache.{name} is fixed when the cache is made" + (": fill it in place" if name in ("pages", "page_table") else ""))
        super().__setattr__(name, value)

    def __init__(self, dtype: GgmlDType, batch: int, kv_heads: int, max_seq: int, head_dim: int, device: torch.device | str = "cuda:0",
                 page_size: Optional[int] = None, num_pages: Optional[int] = None):
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
        self.page_table = torch.full((batch, -(-max_seq // self.page_size)), -1, dtype=torch.int32, device=self.device) if paged else None
        self._view = _Cache(int(self.dtype), kv_heads, head_dim, self.page_size, self.num_pages, self.pages.data_ptr(),
                            self.page_table.data_ptr() if paged else None, self.page_table.stride(0) if paged else 0, max_seq)

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

    def store(self, k: torch.Tensor, v: torch.Tensor, pos: torch.Tensor) -> None:
        """Quantize ``k`` and ``v`` ``[batch, seq, kv_heads, head_dim]`` (f32 / f16 / bf16, any strides) into positions ``pos ..``: the blocks that
        ``BlockQ4_0`` / ``BlockQ8_0::from_float`` make of the f32 values (k_quants.rs:235-270, 636-661), Q8_0's scale being ``max|x| * float32(1 / 127)``."""
        if self._native.kv_store(self._handle, k, v, pos):
            return
        _refuse_derivatives("store", k, v)
        self._tokens("k", k, self.kv_heads), self._tokens("v", v, self.kv_heads)
        if k.shape != v.shape or k.dtype is not v.dtype:
            raise ValueError(f"k is {tuple(k.shape)} {k.dtype}, v {tuple(v.shape)} {v.dtype}")
        self._store(k, v, pos, None)

    def rope_store(self, qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, pos: torch.Tensor, heads: int, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """``qkv`` ``[batch, seq, (heads + 2 kv_heads) * head_dim]``, a fused projection's output: q and k rotated (rotate-half, f32 tables ``[rows, head_dim /
        2]``) at their positions, k and v stored. Returns q ``[batch, seq, heads, head_dim]`` as ``out_dtype`` (default: ``qkv``'s)."""
        if out_dtype is None or out_dtype in _TORCH_TO_XNQ:
            q = self._native.kv_rope_store(self._handle, qkv, cos, sin, pos, heads, -1 if out_dtype is None else _XNQ_IDS[out_dtype])
            if q is not None:
                return q
        _refuse_derivatives("rope_store", qkv, cos, sin)
        hd, width = self.head_dim, (heads + 2 * self.kv_heads) * self.head_dim
        if heads < 1 or qkv.dim() != 3 or qkv.shape[2] != width:
            raise ValueError(f"rope_store: qkv is {tuple(qkv.shape)}; {heads} + 2 * {self.kv_heads} heads of {hd}")
        for t in (cos, sin):
            if t.dtype is not torch.float32 or not t.is_contiguous() or t.dim() != 2 or t.shape[1] != hd // 2 or t.shape != cos.shape or t.device != self.device:
                raise ValueError(f"rope_store: tables are contiguous float32 [rows, {hd // 2}] on {self.device}")
        if out_dtype is not None and out_dtype not in _TORCH_TO_XNQ:
            raise ValueError(f"rope_store: queries of type {out_dtype}")
        x = qkv.unflatten(2, (-1, hd))
        if not _served(x):
            x = x.clone(memory_format=torch.contiguous_format)
        self._tokens("qkv", x)
        q, k, v = x.split([heads, self.kv_heads, self.kv_heads], dim=2)
        out = torch.empty((*q.shape,), dtype=out_dtype or qkv.dtype, device=self.device)
        self._store(k, v, pos, _Rope(cos.data_ptr(), sin.data_ptr(), cos.shape[0], heads, _rows(q), _rows(out)))
        return out

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

    def attend(self, q: torch.Tensor, pos: torch.Tensor, causal: bool = True, window: int = 0, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
               lse: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of ``q`` ``[batch, seq, heads, head_dim]`` (f32 / f16 / bf16, any strides) over the cache; ``heads`` is a multiple of ``kv_heads``.

        Query ``i`` of a sequence is at ``p = pos + i`` and sees positions ``j <= p`` (``causal``) or ``j < pos + seq``, with a ``window`` only ``j > p - window``;
        one that sees nothing gives zeros. ``scale``: default ``head_dim ** -0.5``. ``out``: where the result goes (``q``'s shape and type, rows contiguous and
        16-byte aligned). ``lse``: float32 ``[batch, seq, heads]`` that receives the logarithm of the sum of exponentials (-inf: nothing seen)."""
        if out is None and lse is None:
            res = self._native.kv_attend(self._handle, q, pos, causal, window, self.head_dim ** -0.5 if scale is None else scale)
            if res is not None:
                return res
        _refuse_derivatives("attend", q, out, lse)
        self._tokens("q", q)
        heads, seq = q.shape[2], q.shape[1]
        if heads < 1 or heads % self.kv_heads:
            raise ValueError(f"attend: {heads} query heads over {self.kv_heads} KV heads")
        if window < 0:
            raise ValueError(f"attend: window {window}")
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=self.device)
        elif out.shape != q.shape or out.dtype is not q.dtype or out.device != self.device or not _served(out) or any(s == 0 and n > 1 for s, n in zip(out.stride(), out.shape)):
            raise ValueError(f"attend: out is {tuple(out.shape)} {out.dtype}; q is {tuple(q.shape)} {q.dtype}, and rows are contiguous, apart and 16-byte aligned")
        if lse is not None and (lse.shape != q.shape[:3] or lse.dtype is not torch.float32 or lse.device != self.device or not lse.is_contiguous()):
            raise ValueError(f"attend: lse is contiguous float32 {tuple(q.shape[:3])}")
        if not _served(q):
            q = q.clone(memory_format=torch.contiguous_format)
        pp, stride = self._positions(pos)
        L = _lib.lib()
        with torch.cuda.device(self.device):
            ws, lock = _workspace(self.device, max(16, int(L.xnq_kv_attend_workspace_bytes(self.batch, seq, heads, self.kv_heads, self.head_dim))))
            with lock:   # (the interpreter's is free during the call, which may enqueue two kernels)
                rc = L.xnq_kv_attend(ctypes.byref(self._view), ctypes.byref(_rows(q)), ctypes.byref(_rows(out)), None if lse is None else ctypes.c_void_p(lse.data_ptr()),
                                     self.batch, seq, heads, pp, stride, self.head_dim ** -0.5 if scale is None else float(scale), int(causal), int(window),
                                     ctypes.c_void_p(ws.data_ptr()), ws.numel(), _stream_ptr(self.device))
            _lib.check(rc)
        return out

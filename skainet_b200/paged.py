"""Paged KV cache (skn_paged_*): keys and values of many sequences of unequal lengths in pages of fp16, bf16 or 4 bits, appended with the
rotation of their positions, read by causal attention with an optional sliding window and first tokens that stay visible."""
from __future__ import annotations

import ctypes
from typing import Optional

import numpy as np

from . import _ffi
from .tensor import Context, SKN_OK, _check, _ptr, _raise

_IO = {"torch.float32": 0, "torch.bfloat16": 3}
_io_of_dtype = {}                # torch's own objects, as they are met (torch is not imported here)


def _io_of(t) -> int:
    io = _io_of_dtype.get(t.dtype)
    if io is None:
        io = _IO.get(str(t.dtype))
        if io is None:
            raise ValueError("rows are float32 or bfloat16")
        _io_of_dtype[t.dtype] = io
    return io


class PagedBatch:
    """The sequences of one step: page_table [n, max_pages], token_start [n + 1], lengths [n] (int32 on the device: dense torch tensors; they are
    read when a call runs, so the owner may rewrite them in stream order), the rows n_tokens of the step's arrays and max_new, the most new
    tokens of one sequence."""

    def __init__(self, page_table, token_start, lengths, n_tokens: int, max_new: int):
        n = lengths.shape[0]
        for t, shape in ((page_table, (n, page_table.shape[-1])), (token_start, (n + 1,)), (lengths, (n,))):
            if tuple(t.shape) != shape or not str(t.dtype).endswith("int32") or not t.is_contiguous() or not t.is_cuda:
                raise ValueError("page_table [n, max_pages], token_start [n + 1] and lengths [n] are dense int32 device tensors")
        if not page_table.device.index == token_start.device.index == lengths.device.index:
            raise ValueError("page_table, token_start and lengths are on one device")
        self._keep = page_table, token_start, lengths
        self.device = page_table.device.index
        self.n_seqs, self.n_tokens, self.max_new, self.max_pages = n, int(n_tokens), int(max_new), int(page_table.shape[1])
        self._c = _ffi.PagedBatchSpec(n, self.n_tokens, self.max_new, self.max_pages, _ptr(page_table), _ptr(token_start), _ptr(lengths))
        self._ref = ctypes.byref(self._c)


def _int32(a) -> np.ndarray:
    a = np.asarray(a)
    if a.size and (a.dtype.kind not in "biuf" or not (np.floor(a) == a).all() or a.min() < -2 ** 31 or a.max() >= 2 ** 31):
        raise ValueError("page_table, token_start and lengths are numbers of int32")
    return np.ascontiguousarray(a, dtype=np.int32)


def _host_batch(page_table, token_start, lengths, n_tokens):
    table, starts, lens = _int32(page_table), _int32(token_start), _int32(lengths)
    if table.ndim != 2 or lens.shape != (table.shape[0],) or starts.shape != (table.shape[0] + 1,):
        raise ValueError("Shapes do not align.")
    new = int(np.diff(starts.astype(np.int64)).max(initial=0))
    return _ffi.PagedBatchSpec(table.shape[0], n_tokens, max(new, 0), table.shape[1], table.ctypes.data, starts.ctypes.data, lens.ctypes.data), (table, starts, lens)


class PagedKVCache:
    """`n_pages` pages of `page_tokens` tokens, held as "f16", "bf16" or "q4_0" (4 bits and one fp16 scale per 32 head dims).  rot_dims: the
    first dimensions of keys and queries that append turns by the position (rot_pairs "adjacent": 2 i with 2 i + 1, "halves": i with
    i + rot_dims / 2).  pools: (K, V) device memory of pool_bytes() each that the caller owns; by default the cache's own, zeroed.

    append / gather / attend take host arrays (fp32) and wait; the _dev forms take torch CUDA tensors of float32 or bfloat16 and a PagedBatch
    and only enqueue on the context's stream: work on other streams, such as torch's current one, has to be ordered by the caller."""

    DTYPES = {"f16": 1, "bf16": 3, "q4_0": 4}
    PAIRS = {"adjacent": 0, "halves": 1}

    @classmethod
    def _spec(cls, n_pages, page_tokens, n_kv_heads, head_dim, dtype, rot_dims, rot_base, rot_pairs):
        if dtype not in cls.DTYPES:
            raise ValueError("dtype must be 'f16', 'bf16' or 'q4_0'")
        if rot_pairs not in cls.PAIRS:
            raise ValueError("rot_pairs must be 'adjacent' or 'halves'")
        return _ffi.PagedSpec(n_kv_heads, head_dim, page_tokens, cls.DTYPES[dtype], n_pages, rot_dims, cls.PAIRS[rot_pairs], 0, rot_base)

    @classmethod
    def pool_bytes(cls, n_pages: int, page_tokens: int, n_kv_heads: int, head_dim: int, dtype: str = "f16") -> int:
        """bytes of each of the two pools"""
        n, spec = ctypes.c_int64(), cls._spec(n_pages, page_tokens, n_kv_heads, head_dim, dtype, 0, 1.0, "adjacent")
        _check(None, _ffi.lib().skn_paged_pool_bytes(ctypes.byref(spec), ctypes.byref(n)))
        return n.value

    def __init__(self, ctx: Context, n_pages: int, page_tokens: int, n_kv_heads: int, head_dim: int, dtype: str = "f16", *, rot_dims: int = 0,
                 rot_base: float = 10000.0, rot_pairs: str = "adjacent", pools=None):
        self._h = ctypes.c_void_p()
        spec = self._spec(n_pages, page_tokens, n_kv_heads, head_dim, dtype, rot_dims, rot_base, rot_pairs)
        self.ctx, self.dtype = ctx, dtype
        self.n_pages, self.page_tokens, self.n_kv_heads, self.head_dim = n_pages, page_tokens, n_kv_heads, head_dim
        if pools is not None:
            need = self.pool_bytes(n_pages, page_tokens, n_kv_heads, head_dim, dtype)
            if any(p.numel() * p.element_size() < need or not p.is_contiguous() or not p.is_cuda or p.device.index != ctx.device for p in pools):
                raise ValueError(f"a pool is dense memory of the context's device, {need} bytes")
        self._pools = pools
        rc = _ffi.lib().skn_paged_create(ctx.handle, ctypes.byref(spec), *(map(_ptr, pools) if pools is not None else (None, None)), ctypes.byref(self._h))
        if rc != SKN_OK:
            self._h = ctypes.c_void_p()
            _raise(ctx.handle, rc)
        self._lib = _ffi.lib()
        self._scale = 1.0 / float(np.sqrt(head_dim))

    @property
    def handle(self):
        return self._h

    # ---- host arrays ------------------------------------------------------------------------------------------------------
    def _rows(self, a, heads=None):
        a = np.ascontiguousarray(a, dtype=np.float32)
        if a.ndim != 3 or a.shape[2] != self.head_dim or (heads is not None and a.shape[1] != heads):
            raise ValueError("Shapes do not align.")
        return a

    def append(self, k, v, page_table, token_start, lengths, q=None) -> Optional[np.ndarray]:
        """k, v [n_tokens, n_kv_heads, head_dim]; q [n_tokens, n_q_heads, head_dim]: returned rotated"""
        k, v = self._rows(k, self.n_kv_heads), self._rows(v, self.n_kv_heads)
        q = None if q is None else self._rows(q)
        if v.shape != k.shape or (q is not None and q.shape[0] != k.shape[0]):
            raise ValueError("Shapes do not align.")
        b, keep = _host_batch(page_table, token_start, lengths, k.shape[0])
        out = None if q is None else q.copy()
        _check(self.ctx.handle, self._lib.skn_paged_append(self._h, ctypes.byref(b), k.ctypes.data, v.ctypes.data, _ptr(q), 0 if q is None else q.shape[1], _ptr(out)))
        del keep
        return out

    def gather(self, page_table, token_start, lengths, n_tokens: Optional[int] = None):
        """(K, V) [n_tokens, n_kv_heads, head_dim] of the cached rows at the step's positions (all tokens where token_start counts all); rows
        of nobody are zero"""
        n = int(np.asarray(token_start)[-1]) if n_tokens is None else n_tokens
        b, keep = _host_batch(page_table, token_start, lengths, n)
        k, v = (np.zeros((n, self.n_kv_heads, self.head_dim), dtype=np.float32) for _ in range(2))
        _check(self.ctx.handle, self._lib.skn_paged_gather(self._h, ctypes.byref(b), k.ctypes.data, v.ctypes.data))
        del keep
        return k, v

    def attend(self, q, page_table, token_start, lengths, scale: Optional[float] = None, window: int = 0, sinks: int = 0) -> np.ndarray:
        """q [n_tokens, n_q_heads, head_dim] (rotated) -> outputs of the same shape; rows of nobody are zero"""
        q = self._rows(q)
        b, keep = _host_batch(page_table, token_start, lengths, q.shape[0])
        out = np.zeros_like(q)
        _check(self.ctx.handle, self._lib.skn_paged_attn(self._h, ctypes.byref(b), q.ctypes.data, q.shape[1], self._scale if scale is None else scale, window, sinks,
                                                        out.ctypes.data))
        del keep
        return out

    # ---- device tensors -----------------------------------------------------------------------------------------------------
    def _row_stride(self, t, dtype, n: int, heads: int) -> int:
        """elements between the rows of a device tensor [n, heads, head_dim] whose rows are dense"""
        D, stride = self.head_dim, t.stride()
        if t.dtype is not dtype or t.get_device() != self.ctx.device or tuple(t.shape) != (n, heads, D) or stride[2] != 1 or (stride[1] != D and heads > 1):
            raise ValueError("Shapes do not align." if t.dtype is dtype and t.get_device() == self.ctx.device
                             else "the step's tensors are on the context's device and of one type")
        return stride[0] if n > 1 else heads * D

    def append_dev(self, batch: PagedBatch, k, v, q=None, q_out=None):
        """rows may be parts of wider ones (a joint projection); q_out is q or lies elsewhere; its rows of nobody and padded rows stay as they are"""
        io, n, kv, dt, row = _io_of(k), batch.n_tokens, self.n_kv_heads, k.dtype, self._row_stride
        if batch.device != self.ctx.device:
            raise ValueError("the step's tensors are on the context's device and of one type")
        if q is None:
            more = (None, 0, 0, None, 0)
        else:
            if q_out is None:
                raise ValueError("the rotated queries need q_out (which may be q)")
            heads = q.shape[1]
            more = (q.data_ptr(), row(q, dt, n, heads), heads, q_out.data_ptr(), row(q_out, dt, n, heads))
        rc = self._lib.skn_paged_append_dev(self._h, batch._ref, io, k.data_ptr(), row(k, dt, n, kv), v.data_ptr(), row(v, dt, n, kv), *more)
        if rc:
            _raise(self.ctx.handle, rc)

    def gather_dev(self, batch: PagedBatch, k_out, v_out):
        io, shape = _io_of(k_out), (batch.n_tokens, self.n_kv_heads, self.head_dim)
        if batch.device != self.ctx.device or any(t.get_device() != self.ctx.device or t.dtype is not k_out.dtype for t in (k_out, v_out)):
            raise ValueError("the step's tensors are on the context's device and of one type")
        if k_out.shape != shape or v_out.shape != shape or not k_out.is_contiguous() or not v_out.is_contiguous():
            raise ValueError("Shapes do not align.")
        rc = self._lib.skn_paged_gather_dev(self._h, batch._ref, io, k_out.data_ptr(), v_out.data_ptr())
        if rc:
            _raise(self.ctx.handle, rc)

    def attend_dev(self, batch: PagedBatch, q, out, scale: Optional[float] = None, window: int = 0, sinks: int = 0):
        """q [n_tokens, n_q_heads, head_dim] (rotated) -> out, which may lie beside q in wider rows, but not over it; rows of nobody stay as they are"""
        io, n, heads, row = _io_of(q), batch.n_tokens, q.shape[1], self._row_stride
        if batch.device != self.ctx.device:
            raise ValueError("the step's tensors are on the context's device and of one type")
        rc = self._lib.skn_paged_attn_dev(self._h, batch._ref, io, q.data_ptr(), row(q, q.dtype, n, heads), heads, self._scale if scale is None else scale,
                                          window, sinks, out.data_ptr(), row(out, q.dtype, n, heads))
        if rc:
            _raise(self.ctx.handle, rc)

    def close(self):
        if self._h:
            _ffi.lib().skn_paged_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

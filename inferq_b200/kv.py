"""A paged key/value cache on the device and the attention over it (the
``iq_kv_*`` part of include/iq.h).

    cache = KvCache(kv_heads=2, head_dim=256, pages=4096, page_tokens=64, format="i8")
    batch = KvBatch(table, position, row_start, max_rows=4)   # int32 CUDA tensors
    cache.append(k, v, batch)                                 # [rows, kv_heads, head_dim]
    out = cache.attend(q, batch)                              # [rows, heads, head_dim]
    k, v = cache.read(batch, dtype=torch.float32, rows=8)

One ``KvCache`` holds one layer.  Calls are enqueued on the current stream of
the cache's device unless ``stream`` (a handle) is given; the tensors of such a
call may be let go at once.
"""
from __future__ import annotations

import ctypes
import sys

import torch

from . import _lib

F16, I8 = 1, 24
FORMATS = {"f16": F16, "i8": I8}
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}

P, I64, I32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int

_KEPT = 64  # argument structures that a batch or a cache keeps for calls like earlier ones


class _Batch(ctypes.Structure):
    _fields_ = [("table", P), ("position", P), ("row_start", P), ("table_ld", I64), ("table_cols", ctypes.c_int32),
                ("seqs", ctypes.c_int32), ("rows", ctypes.c_int32), ("max_rows", ctypes.c_int32)]


class _Attn(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int32), ("heads", ctypes.c_int32), ("scale", ctypes.c_float),
                ("window", ctypes.c_int32), ("sinks", ctypes.c_int32), ("chunk", ctypes.c_int32)]


def _lib_():
    L = _lib.lib()
    if not getattr(L, "_kv_declared", False):
        B, A = ctypes.POINTER(_Batch), ctypes.POINTER(_Attn)
        sig = {
            "iq_kv_create": (I32, [I32, I32, I32, I32, I64, ctypes.POINTER(P)]),
            "iq_kv_destroy": (None, [P]),
            "iq_kv_bytes": (I32, [P, ctypes.POINTER(I64)]),
            "iq_kv_append": (I32, [P, B, I32, P, I64, I64, P, I64, I64, P]),
            "iq_kv_read": (I32, [P, B, I32, P, I64, I64, P, I64, I64, P]),
            "iq_kv_attend_workspace": (I32, [P, B, A, ctypes.POINTER(ctypes.c_size_t)]),
            "iq_kv_attend": (I32, [P, B, A, P, I64, I64, P, I64, I64, P, ctypes.c_size_t, P]),
            "iq_kv_status": (I32, [P, P]),
        }
        for n, (r, a) in sig.items():
            f = getattr(L, n)
            f.restype, f.argtypes = r, a
        L._kv_declared = True
    return L


class KvBatch:
    """Rows of several sequences: ``table`` [seqs, columns] int32 page ids,
    ``position`` [seqs] int32 positions of the sequences' first rows, and
    ``row_start`` [seqs + 1] int32 (None: one sequence that owns all rows);
    CUDA tensors.  ``max_rows``: the most rows of one sequence as far as the
    host knows (0: not known); it picks the kernel."""

    def __init__(self, table: torch.Tensor, position: torch.Tensor, row_start: torch.Tensor | None = None, *,
                 max_rows: int = 0):
        for name, x, dims in (("table", table, 2), ("position", position, 1), ("row_start", row_start, 1)):
            if x is None and name == "row_start":
                continue
            if x.dtype != torch.int32 or x.dim() != dims:
                raise ValueError(f"{name} must be an int32 tensor of {dims} dimensions, got {x.dtype} of {x.dim()}")
            if not x.is_cuda or x.device != table.device:
                raise ValueError(f"{name} must be on the CUDA device of the table")
            if x.shape[-1] > 1 and x.stride(-1) != 1:
                raise ValueError(f"{name} must be contiguous along its last dimension")
        seqs = table.shape[0]
        if position.shape[0] != seqs:
            raise ValueError(f"{position.shape[0]} positions for {seqs} block tables")
        if row_start is None and seqs != 1:
            raise ValueError(f"{seqs} sequences need row_start")
        if row_start is not None and row_start.shape[0] != seqs + 1:
            raise ValueError(f"row_start has {row_start.shape[0]} entries for {seqs} sequences")
        if max_rows < 0:
            raise ValueError("max_rows cannot be negative")
        _lib.fits(max_rows=max_rows)
        self.device, self.index = table.device, table.get_device()
        self.seqs = seqs
        self._keep = table, position, row_start
        ld = table.stride(0) if seqs > 1 else max(table.stride(0), table.shape[1])
        self._c = _Batch(table.data_ptr(), position.data_ptr(), None if row_start is None else row_start.data_ptr(), ld,
                         table.shape[1], seqs, 0, max_rows)
        self._of_rows: dict[int, _Batch] = {}

    def _with(self, rows: int) -> _Batch:
        got = self._of_rows.get(rows)
        if got is None:
            c = self._c
            got = _Batch(c.table, c.position, c.row_start, c.table_ld, c.table_cols, c.seqs, rows, c.max_rows)
            if len(self._of_rows) >= _KEPT:
                self._of_rows.clear()
            self._of_rows[rows] = got
        return got


# Caches let go of while a stream was captured, freed when the next is made or let go.
_dropped: list[tuple] = []


def _free_dropped():
    while _dropped:
        device, h = _dropped.pop()
        try:
            torch.cuda.synchronize(device)
        except RuntimeError:  # (another thread captures)
            _dropped.append((device, h))
            return
        _lib._lib.iq_kv_destroy(h)


class KvCache:
    """One layer's paged cache on ``device`` (default: the current one)."""

    def __init__(self, kv_heads: int, head_dim: int, pages: int, *, page_tokens: int = 64, format: str = "i8",
                 device=None):
        if format not in FORMATS:
            raise ValueError(f"cache format {format!r}; expected one of {sorted(FORMATS)}")
        _lib.fits(kv_heads=kv_heads, head_dim=head_dim, page_tokens=page_tokens)
        _lib.fits(64, pages=pages)
        self.kv_heads, self.head_dim, self.pages, self.page_tokens = kv_heads, head_dim, pages, page_tokens
        self.format = format
        self._lib = _lib_()
        _free_dropped()
        h = P()
        dev = torch.device("cuda" if device is None else device)
        with torch.cuda.device(dev):
            _lib.check(self._lib.iq_kv_create(FORMATS[format], kv_heads, head_dim, page_tokens, pages, ctypes.byref(h)))
            self.device = torch.device("cuda", torch.cuda.current_device())
        self._h = h
        self._index = self.device.index
        self._attn: dict[tuple, _Attn] = {}

    @property
    def nbytes(self) -> int:
        n = I64()
        _lib.check(self._lib.iq_kv_bytes(self._h, ctypes.byref(n)))
        return n.value

    def _stream(self, stream):
        # (the handle alone: current_stream() builds a stream object, 2 us a call)
        return torch._C._cuda_getCurrentRawStream(self._index) if stream is None else stream

    def _new(self, shape, dtype, stream):
        """Memory of the stream that writes it; the current one may read it."""
        with torch.cuda.stream(torch.cuda.ExternalStream(stream, device=self.device)):
            x = torch.empty(shape, dtype=dtype, device=self.device)
        if x.numel():
            x.record_stream(torch.cuda.current_stream(self.device))
        return x

    def _on(self, stream, batch, *tensors):
        """The stream for a call on ``tensors``; one given by handle reads (or
        writes) them and the batch after the caller may have let them go."""
        if stream is None:
            return self._stream(None)
        st = torch.cuda.ExternalStream(stream, device=self.device)
        for x in (*tensors, *batch._keep):
            if x is not None and x.numel():
                x.record_stream(st)
        return stream

    def _rows(self, name, x, heads, batch):
        shape = x.shape
        if x.dtype not in _TYPES:
            raise ValueError(f"{name} must be float32, float16 or bfloat16, got {x.dtype}")
        if x.get_device() != self._index or batch.index != self._index:
            raise ValueError(f"{name} and the batch must be on the cache's device {self.device}")
        if len(shape) != 3 or shape[2] != self.head_dim or (heads and shape[1] != heads):
            raise ValueError(f"{name} must be [rows, {heads or 'heads'}, {self.head_dim}], got {list(shape)}")
        row, head, elt = x.stride()
        if elt != 1:
            raise ValueError(f"the elements of a head of {name} must be contiguous")
        return x.data_ptr(), row, head

    def append(self, k: torch.Tensor, v: torch.Tensor, batch: KvBatch, *, stream=None) -> None:
        """Quantise rows [rows, kv_heads, head_dim] into the cache."""
        if k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("keys and values must have one shape and type")
        a, b = self._rows("keys", k, self.kv_heads, batch), self._rows("values", v, self.kv_heads, batch)
        _lib.check(self._lib.iq_kv_append(self._h, batch._with(k.shape[0]), _TYPES[k.dtype], *a, *b,
                                          self._on(stream, batch, k, v)))

    def read(self, batch: KvBatch, *, rows: int, dtype=torch.float32, out=None, stream=None):
        """(keys, values) that the cache holds at the batch's ``rows`` rows;
        rows behind the last sequence are left as they are in ``out``."""
        if out is None:
            shape = (rows, self.kv_heads, self.head_dim)
            if stream is None:
                out = (torch.empty(shape, dtype=dtype, device=self.device),
                       torch.empty(shape, dtype=dtype, device=self.device))
            else:
                out = self._new(shape, dtype, stream), self._new(shape, dtype, stream)
        k, v = out
        if k.shape != v.shape or k.dtype != v.dtype or k.shape[0] != rows:
            raise ValueError("keys and values must have one shape and type, and the batch's rows")
        a, b = self._rows("keys", k, self.kv_heads, batch), self._rows("values", v, self.kv_heads, batch)
        _lib.check(self._lib.iq_kv_read(self._h, batch._with(rows), _TYPES[k.dtype], *a, *b,
                                        self._on(stream, batch, k, v)))
        return k, v

    def attend(self, q: torch.Tensor, batch: KvBatch, *, scale: float = 0.0, window: int = 0, sinks: int = 0,
               chunk: int = 0, out=None, stream=None) -> torch.Tensor:
        """Causal attention of rows ``q`` [rows, heads, head_dim] over their
        sequences' cached tokens (which include the rows' own: append first);
        see iq_kv_attend for ``window``, ``sinks``, ``scale`` and ``chunk``."""
        a = self._rows("queries", q, 0, batch)
        rows, heads, _ = q.shape
        if out is None:
            # (empty_like: a microsecond less than torch.empty)
            out = (torch.empty_like(q, memory_format=torch.contiguous_format) if stream is None else
                   self._new(q.shape, q.dtype, stream))
        elif out.shape != q.shape or out.dtype != q.dtype:
            raise ValueError("queries and outputs must have one shape and type")
        b = self._rows("outputs", out, heads, batch)
        key = q.dtype, heads, scale, window, sinks, chunk
        at = self._attn.get(key)
        if at is None:
            _lib.fits(window=window, sinks=sinks, chunk=chunk)
            if len(self._attn) >= _KEPT:
                self._attn.clear()
            at = self._attn[key] = _Attn(_TYPES[q.dtype], heads, scale, window, sinks, chunk)
        c, need = batch._with(rows), ctypes.c_size_t()
        _lib.check(self._lib.iq_kv_attend_workspace(self._h, c, at, need))
        ws, n = None, need.value
        if n:
            ws = q.new_empty(n, dtype=torch.uint8) if stream is None else self._new(n, torch.uint8, stream)
        _lib.check(self._lib.iq_kv_attend(self._h, c, at, *a, *b, None if ws is None else ws.data_ptr(), n,
                                          self._on(stream, batch, q, out)))
        return out

    def status(self, stream=None) -> None:
        """Synchronise ``stream`` and raise IqError if a call on this cache met
        a position or page id out of range (or gave up a device wait)."""
        _lib.check(self._lib.iq_kv_status(self._h, self._stream(stream)))

    def __del__(self):
        h = getattr(self, "_h", None)
        if h is None or sys is None or sys.is_finalizing():  # (the process's end frees it)
            return
        self._h = None
        _dropped.append((self.device, h))
        if not torch.cuda.is_current_stream_capturing():  # neither waiting nor freeing may be captured: later then
            _free_dropped()

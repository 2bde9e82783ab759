"""Python binding of the paged-cache operators (ill_paged_* in include/ill_hip.h): new rows into
a paged key/value cache, and attention over it, for several sequences at once.

As in `Gemv.run_noalloc`, buffers are device addresses that the caller owns, work is enqueued on
the caller's stream (None: the default one), nothing is allocated and nothing waited for.
"""
from __future__ import annotations

import ctypes as C
import struct

from .engine import ILL_OK, IllError, load_library

DTYPES = {"f32": 0, "f16": 1, "bf16": 2}


class _Desc(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("dtype", "heads", "kv_heads", "head_dim", "page_size", "rotary_dim", "interleaved", "streams")] + \
               [(n, C.c_int64) for n in ("page_stride", "slot_stride", "head_stride")] + \
               [("rope_base", C.c_double), ("norm_eps", C.c_float), ("scale", C.c_float)]


class Batch(C.Structure):
    """The sequences of a call (ill_paged_batch); the arrays are read when the kernels run."""
    _fields_ = [("seqs", C.c_int32), ("table_width", C.c_int32)] + \
               [(n, C.c_int64) for n in ("table_stride", "rows", "max_rows", "pages")] + [(n, C.c_void_p) for n in ("lens", "table", "row0")]


class _Rows(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("q", "k", "v", "q_out")] + [(n, C.c_int64) for n in ("q_stride", "k_stride", "v_stride", "q_out_stride")] + \
               [(n, C.c_void_p) for n in ("bias", "q_norm", "k_norm", "positions")] + [("dtype", C.c_int32), ("reserved", C.c_int32)]


# a Batch and a _Rows, faster than field by field; numbers that do not fit are an error (ctypes cuts them off)
_pack_batch = struct.Struct("iiqqqqPPP").pack
_pack_rows = struct.Struct("PPPPqqqqPPPPii").pack


def _fits(bits: int, **values: int):
    for name, v in values.items():
        if not -1 << bits - 1 <= v < 1 << bits - 1:
            raise ValueError(f"{name} {v}: more than {bits} bits")


def _dtype(name: str) -> int:
    if name not in DTYPES:
        raise ValueError(f"type {name!r}: one of {', '.join(DTYPES)}")
    return DTYPES[name]


class PagedAttention:
    """A model's head geometry and cache layout. `strides`: (page, slot, head) strides of the
    caches in elements (None: [pages][page_size][kv_heads][head_dim]); `rotary_dim` None: the
    whole head; `streams`: how many streams, and captures of streams, attention calls may come on."""

    def __init__(self, heads: int, kv_heads: int, head_dim: int, page_size: int = 16, dtype: str = "f16", rotary_dim: int | None = None,
                 rope_base: float = 1e6, interleaved: bool = False, norm_eps: float = 1e-6, scale: float | None = None,
                 strides: tuple[int, int, int] | None = None, streams: int = 8):
        self.h = None
        self.lib = load_library()
        self.heads, self.kv_heads, self.head_dim, self.dtype, self.type = heads, kv_heads, head_dim, dtype, _dtype(dtype)
        self.q_width, self.kv_width = heads * head_dim, kv_heads * head_dim
        _fits(32, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page_size=page_size, rotary_dim=rotary_dim or 0, streams=streams)
        _fits(64, **dict(zip(("page_stride", "slot_stride", "head_stride"), strides or ())))
        d = _Desc(self.type, heads, kv_heads, head_dim, page_size, head_dim if rotary_dim is None else rotary_dim, int(interleaved), streams,
                  *(strides or (0, 0, 0)), rope_base, norm_eps, scale or 0.0)
        h = C.c_void_p()
        self._check(self.lib.ill_paged_create(C.byref(d), C.byref(h)))
        self.h = h

    def _check(self, rc: int):
        if rc != ILL_OK:
            raise IllError(rc, self.lib.ill_last_error().decode())

    def batch(self, lens: int, table: int, table_width: int, pages: int, seqs: int, rows: int | None = None, row0: int | None = None,
              max_rows: int = 0, table_stride: int | None = None) -> Batch:
        """lens [seqs], table [seqs][table_stride], row0 [seqs + 1] (None: one row each): device addresses of int32 arrays."""
        try:
            return Batch.from_buffer_copy(_pack_batch(seqs, table_width, table_width if table_stride is None else table_stride, seqs if rows is None else rows,
                                                      max_rows, pages, lens or 0, table or 0, row0 or 0))
        except struct.error as e:
            raise ValueError(f"a batch's sizes and addresses: {e}") from None

    def append(self, batch: Batch, k_cache: int, v_cache: int, k: int, v: int, q: int | None = None, q_out: int | None = None,
               x_dtype: str | None = None, x_stride: int | None = None, q_stride: int | None = None, k_stride: int | None = None,
               v_stride: int | None = None, q_out_stride: int | None = None, bias: int | None = None, q_norm: int | None = None,
               k_norm: int | None = None, positions: int | None = None, stream: int | None = None):
        """New rows into the cache; the turned queries go to q_out. x_dtype None: the cache's. x_stride: the row stride of q, k and
        v, where one is not given; without either, rows are contiguous."""
        qw, kw = self.q_width, self.kv_width
        if x_stride is not None:
            qw = kw = x_stride
        try:
            x = _pack_rows(q or 0, k or 0, v or 0, q_out or 0, qw if q_stride is None else q_stride, kw if k_stride is None else k_stride,
                           kw if v_stride is None else v_stride, self.q_width if q_out_stride is None else q_out_stride, bias or 0, q_norm or 0,
                           k_norm or 0, positions or 0, self.type if x_dtype is None else _dtype(x_dtype), 0)
        except struct.error as e:
            raise ValueError(f"strides and addresses of rows: {e}") from None
        rc = self.lib.ill_paged_append(self.h, C.byref(batch), x, k_cache, v_cache, stream)
        if rc:
            self._check(rc)

    def attend(self, batch: Batch, k_cache: int, v_cache: int, q: int, out: int, out_dtype: str | None = None, window: int = 0, sinks: int = 0,
               q_stride: int | None = None, out_stride: int | None = None, stream: int | None = None):
        """Attention of the new rows over the cache, all earlier positions or the last `window` and the first `sinks`."""
        q_stride, out_stride = self.q_width if q_stride is None else q_stride, self.q_width if out_stride is None else out_stride
        if (window | sinks) >> 31 or (q_stride | out_stride) >> 31:   # (negative ones are the library's to refuse)
            _fits(32, window=window, sinks=sinks)
            _fits(64, q_stride=q_stride, out_stride=out_stride)
        rc = self.lib.ill_paged_attend(self.h, C.byref(batch), q, q_stride, k_cache, v_cache, window, sinks, out, out_stride,
                                       self.type if out_dtype is None else _dtype(out_dtype), stream)
        if rc:
            self._check(rc)

    def bind(self, stream: int | None, workspace: int | None):
        """Calls on the stream, captured or not, take this of the `streams` workspaces from now on: streams that never run at the same
        time, and graphs launched in order, may share one. None: the stream's workspaces are free (when nothing that came on
        it will run any more, and before it is destroyed)."""
        w = -1 if workspace is None else workspace
        _fits(32, workspace=w)
        self._check(self.lib.ill_paged_bind(self.h, stream, w))

    def release(self):
        """Frees the workspaces of all streams and captures (when nothing enqueued or captured will run any more)."""
        self._check(self.lib.ill_paged_release(self.h))

    def close(self):
        if getattr(self, "h", None):
            self.lib.ill_paged_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

"""Python binding of the microscaled operators (ill_mx_* in include/ill_hip.h): rows of blocks of 32 values that share a power of
two, in 8 or 4 bits a value, and products with matrices of 4 bits a value.

As in `paged.PagedAttention`, buffers are device addresses that the caller owns, work is enqueued on the caller's stream (None: the
default one), nothing is allocated and nothing waited for.
"""
from __future__ import annotations

from .engine import ILL_OK, IllError, load_library

DTYPES = {"f32": 0, "f16": 1, "bf16": 2}
FORMATS = {"mxf8": 8, "mxf4": 16}
BLOCK = 32   # values that share a power


def _one_of(what: str, name: str, of: dict[str, int]) -> int:
    if name not in of:
        raise ValueError(f"{what} {name!r}: one of {', '.join(of)}")
    return of[name]


def _fits(**values: int):   # (ctypes cuts numbers off; asked where one of them is large or negative: those are the library's to refuse)
    for name, v in values.items():
        if not -1 << 63 <= v < 1 << 63:
            raise ValueError(f"{name} {v}: more than 64 bits")


def _check(rc: int):
    if rc != ILL_OK:
        raise IllError(rc, load_library().ill_last_error().decode())


def code_bytes(format: str, values: int) -> int:
    """Bytes of so many values' codes; their powers take values / 32 more, in an array of their own."""
    return values if _one_of("format", format, FORMATS) == FORMATS["mxf8"] else values // 2


def quantize(x: int, codes: int, powers: int, rows: int, cols: int, format: str = "mxf8", dtype: str = "f16", x_stride: int | None = None,
             stream: int | None = None):
    """x [rows][cols] of type dtype to codes and powers."""
    x_stride = cols if x_stride is None else x_stride
    if (rows | cols | x_stride) >> 62:
        _fits(rows=rows, cols=cols, x_stride=x_stride)
    rc = load_library().ill_mx_quantize(_one_of("format", format, FORMATS), _one_of("type", dtype, DTYPES), x, x_stride, rows, cols, codes, powers, stream)
    if rc:
        _check(rc)


def dequantize(codes: int, powers: int, y: int, rows: int, cols: int, format: str = "mxf8", dtype: str = "f16", y_stride: int | None = None,
               stream: int | None = None):
    """codes and powers to values y [rows][cols] of type dtype."""
    y_stride = cols if y_stride is None else y_stride
    if (rows | cols | y_stride) >> 62:
        _fits(rows=rows, cols=cols, y_stride=y_stride)
    rc = load_library().ill_mx_dequantize(_one_of("format", format, FORMATS), _one_of("type", dtype, DTYPES), codes, powers, rows, cols, y, y_stride, stream)
    if rc:
        _check(rc)


def product(x: int, x_powers: int, w: int, w_powers: int, y: int, rows: int, cols: int, inner: int, format: str = "mxf8", dtype: str = "f16",
            bias: int | None = None, y_stride: int | None = None, stream: int | None = None):
    """y [rows][cols] of type dtype: microscaled rows x [rows][inner] of the format times the rows of w [cols][inner], of format
    mxf4, plus bias [cols] (float32)."""
    y_stride = cols if y_stride is None else y_stride
    if (rows | cols | inner | y_stride) >> 62:
        _fits(rows=rows, cols=cols, inner=inner, y_stride=y_stride)
    rc = load_library().ill_mx_product(_one_of("format", format, FORMATS), x, x_powers, w, w_powers, rows, cols, inner, bias,
                                       _one_of("type", dtype, DTYPES), y, y_stride, stream)
    if rc:
        _check(rc)

"""Float64 restatement of the microscaled operators as include/ill_hip.h defines them: blocks of 32 values that share a power of
two. Formats: "mxf8" (e4m3 codes) and "mxf4" (e2m1, two to a byte)."""
from __future__ import annotations

import numpy as np

E4M3 = np.array([(1 + m / 8) * 2.0 ** (e - 7) if e else m / 8 * 2.0 ** -6 for e in range(16) for m in range(8)][:127])   # (the last one is NaN)
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
SIZES = {"mxf8": E4M3, "mxf4": E2M1}
TOP = {"mxf8": 8, "mxf4": 2}   # the largest code's exponent


def pack(codes: np.ndarray, fmt: str) -> np.ndarray:
    """Codes, one to an element, as they lie in memory."""
    return codes.astype(np.uint8) if fmt == "mxf8" else (codes[..., ::2] | codes[..., 1::2] << 4).astype(np.uint8)


def unpack(held: np.ndarray, fmt: str) -> np.ndarray:
    return held if fmt == "mxf8" else np.stack((held & 15, held >> 4), -1).reshape(*held.shape[:-1], -1)


def quantize(x: np.ndarray, fmt: str) -> tuple[np.ndarray, np.ndarray]:
    """x [..., n] to (codes as they lie in memory, power bytes [..., n / 32])."""
    block = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 32)
    sizes, top = SIZES[fmt], TOP[fmt]
    sign = {"mxf8": 128, "mxf4": 8}[fmt]
    bad = ~np.isfinite(block).all(-1)
    most = np.where(bad, 1, np.abs(np.where(np.isfinite(block), block, 0)).max(-1))
    power = np.maximum(np.frexp(most)[1] - 1 - top, -127)
    power = np.where(most == 0, -127, power)
    y = np.minimum(np.ldexp(np.where(bad[..., None], 0, np.abs(block)), -power[..., None]), sizes[-1])
    hi = np.minimum(np.searchsorted(sizes, y), len(sizes) - 1)
    lo = np.maximum(hi - 1, 0)
    below, above = y - sizes[lo], sizes[hi] - y
    code = np.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
    code = np.where(bad[..., None], 0, code + sign * np.signbit(block))
    return pack(code.reshape(x.shape), fmt), np.where(bad, 255, power + 127).astype(np.uint8)


def values(held: np.ndarray, powers: np.ndarray, fmt: str) -> np.ndarray:
    codes = unpack(held, fmt).astype(np.int64)
    sign = {"mxf8": 128, "mxf4": 8}[fmt]
    size = np.append(E4M3, np.nan)[codes & 127] if fmt == "mxf8" else E2M1[codes & 7]
    y = np.where(codes & sign, -size, size).reshape(*powers.shape, 32)
    scale = np.where(powers == 255, np.nan, np.ldexp(1.0, powers.astype(np.int64) - 127))
    with np.errstate(invalid="ignore"):
        return (y * scale[..., None]).reshape(codes.shape)


def held_as(y: np.ndarray, powers: np.ndarray, fmt: str) -> np.ndarray:
    """The values that y [..., n] is held as in blocks of these power bytes [..., n / 32]: nearest, ties to the even code."""
    sizes = SIZES[fmt]
    scale = np.ldexp(1.0, powers.astype(np.int64) - 127)[..., None]
    z = np.minimum(np.abs(np.asarray(y, np.float64).reshape(*powers.shape, 32)) / scale, sizes[-1])
    hi = np.minimum(np.searchsorted(sizes, z), len(sizes) - 1)
    lo = np.maximum(hi - 1, 0)
    below, above = z - sizes[lo], sizes[hi] - z
    code = np.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
    return (np.copysign(sizes[code], np.reshape(y, (*powers.shape, 32))) * scale).reshape(np.shape(y))

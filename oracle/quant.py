"""The 8-bit row format of the quantised KV cache, on numpy arrays.

A row x[0..127] of one (token, KV head) with finite maximum a = m * 2^E, 1 <= m < 2, is
kept as the power of two 2^e, e = max(E - 8 + (m > 1.75), -117), and the codes
e4m3(x_i * 2^-e), rounded to nearest even; NaN and infinities become NaN.
Everything is computed with integers and exact float64 operations: e4m3 has four
significant bits, exponents from -6 (steps of 2^-9 below it) and 448 as its maximum.
"""
from __future__ import annotations

import numpy as np

PAGE = 256
D = 128
RECORD = PAGE * D + PAGE


def scale_exponent(x: np.ndarray) -> np.ndarray:
    """e of rows [..., 128] (float64 holding bf16 values)."""
    x = np.asarray(x, dtype=np.float64)
    a = np.where(np.isfinite(x), np.abs(x), 0.0).max(-1)
    frac, exp = np.frexp(a)  # a = frac * 2^exp, frac in [0.5, 1)
    e = exp - 1 - 8 + (2 * frac > 1.75)
    return np.where(a > 0, np.maximum(e, -117), -117).astype(np.int64)


def encode(y: np.ndarray) -> np.ndarray:
    """e4m3 codes (uint8) of float64 values with |y| <= 448; NaN and infinities -> 0x7f."""
    y = np.asarray(y, dtype=np.float64)
    ok = np.isfinite(y)
    v = np.where(ok, y, 0.0)
    _, exp = np.frexp(v)
    e = np.maximum(np.where(v == 0, -6, exp - 1), -6)
    n = np.rint(np.abs(v) / np.ldexp(1.0, e - 3)).astype(np.int64)  # steps of 2^(e-3); rint: ties to even
    # n in 0 .. 16: 16 carries into the next exponent, below 8 the value is subnormal
    code = np.where(n < 8, n, ((e + 7) << 3) + (n - 8))
    code = np.where(np.signbit(v), code | 0x80, code)
    return np.where(ok, code, 0x7F).astype(np.uint8)


def decode(code: np.ndarray) -> np.ndarray:
    """float64 values of e4m3 codes."""
    c = np.asarray(code, dtype=np.int64)
    mant, exp = c & 7, (c >> 3) & 15
    v = np.where(exp == 0, mant * 2.0 ** -9, (8 + mant) * np.ldexp(1.0, exp - 10))
    v = np.where((c & 0x7F) == 0x7F, np.nan, v)
    return np.where(c & 0x80, -v, v)


def quantise(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """(codes [..., 128], scale bytes [...]) of rows of bf16 values."""
    e = scale_exponent(x)
    return encode(np.asarray(x, dtype=np.float64) * np.ldexp(1.0, -e)[..., None]), (e + 127).astype(np.uint8)


def dequantise(codes: np.ndarray, scale: np.ndarray) -> np.ndarray:
    """float64 values; from 2^128 on they are infinite in bf16."""
    v = decode(codes) * np.ldexp(1.0, scale.astype(np.int64) - 127)[..., None]
    return np.where(np.abs(v) >= 2.0 ** 128, np.copysign(np.inf, v), v)


def store(rows: np.ndarray, pages: np.ndarray, slots) -> None:
    """rows [N, H, 128] into pages (uint8 [P, H, RECORD]) by slot; slots outside are skipped."""
    codes, scale = quantise(rows)
    for i, s in enumerate(np.asarray(slots).reshape(-1).tolist()):
        if 0 <= s < pages.shape[0] * PAGE:
            p, r = divmod(s, PAGE)
            pages[p, :, r * D:(r + 1) * D] = codes[i]
            pages[p, :, PAGE * D + r] = scale[i]


def load(pages: np.ndarray, slots) -> np.ndarray:
    """Rows [N, H, 128] (float64) that slots inside the cache hold."""
    out = []
    for s in np.asarray(slots).reshape(-1).tolist():
        p, r = divmod(s, PAGE)
        out.append(dequantise(pages[p, :, r * D:(r + 1) * D], pages[p, :, PAGE * D + r]))
    return np.stack(out) if out else np.zeros((0, pages.shape[1], D))

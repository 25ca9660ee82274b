"""CPU restatement of the block-scaled cache formats in float64 (test
infrastructure only): groups of 32 elements under a power-of-two scale,
elements E2M1 ("fp4") or E4M3 ("fp8"). include/skv.h states the rule.
"""
from __future__ import annotations

import numpy as np

GROUP = 32
_E = {"fp4": (7.0, -100, 125), "fp8": (464.0, -100, 119)}


def grid(fmt: str) -> np.ndarray:
    """Non-negative element values in code order."""
    man, bias, n = (1, 1, 8) if fmt == "fp4" else (3, 7, 127)
    code = np.arange(n)
    e, m = code >> man, code & ((1 << man) - 1)
    return np.where(e == 0, np.ldexp(m, 1 - bias - man), np.ldexp((1 << man) + m, e - bias - man))


def quantise(x: np.ndarray, fmt: str) -> tuple[np.ndarray, np.ndarray]:
    """(codes, one to a byte, of x's shape; scale bytes [..., d / 32])."""
    x = np.asarray(x, np.float64)
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    top, lo, hi = _E[fmt]
    with np.errstate(invalid="ignore"):
        amax = np.abs(g).max(-1)
    bad = ~np.isfinite(amax)
    e = np.full(amax.shape, lo, np.int64)
    pos = ~bad & (amax > 0)
    # top 2^(e-1) < amax <= top 2^e: amax / top = m 2^p with m in [1/2, 1)
    ratio_m, ratio_p = np.frexp(amax[pos])
    tm, tp = np.frexp(top)
    e[pos] = ratio_p - tp + (ratio_m > tm)
    e = np.clip(e, lo, hi)
    gr = grid(fmt)
    with np.errstate(invalid="ignore"):
        y = np.abs(np.ldexp(g, -e[..., None]))
    y = np.minimum(np.where(np.isfinite(y), y, 0.0), gr[-1])
    mid = (gr[1:] + gr[:-1]) / 2
    low, high = np.searchsorted(mid, y, "left"), np.searchsorted(mid, y, "right")
    code = np.where(low % 2 == 0, low, high)  # on a midpoint: the even code
    code = code + np.where(np.signbit(g), 8 if fmt == "fp4" else 128, 0)
    code = np.where(bad[..., None], 0, code).astype(np.uint8)
    byte = np.where(bad, 255, e + 127).astype(np.uint8)
    return code.reshape(x.shape), byte


def values(code: np.ndarray, byte: np.ndarray, fmt: str) -> np.ndarray:
    """The float64 values of codes [..., d] under scale bytes [..., d / 32]."""
    half = 8 if fmt == "fp4" else 128
    gr = np.append(grid(fmt), np.nan) if fmt == "fp8" else grid(fmt)
    v = gr[code % half] * np.where(code >= half, -1.0, 1.0)
    s = np.where(byte == 255, np.nan, np.ldexp(1.0, byte.astype(np.int64) - 127))
    return v * np.repeat(s, GROUP, -1)


def round_trip(x: np.ndarray, fmt: str) -> np.ndarray:
    return values(*quantise(x, fmt), fmt)


def pack(code: np.ndarray, fmt: str) -> np.ndarray:
    return code if fmt == "fp8" else code[..., 0::2] | (code[..., 1::2] << 4)


def attention(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float,
              last: np.ndarray) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """One kv head: q [rows, d] over k, v [t, d], row i sees positions <=
    last[i]. (outputs, sum p |v|, max_t sum |q k| scale), the last two for error
    bounds. Rows that see nothing are zeros."""
    out = np.zeros(q.shape)
    mag = np.zeros(q.shape)
    big = np.zeros(q.shape[0])
    for i in range(q.shape[0]):
        n = int(last[i]) + 1
        if n <= 0:
            continue
        s = (k[:n] @ q[i]) * scale
        with np.errstate(invalid="ignore"):
            w = np.exp(s - s.max())
            w = w / w.sum()
        out[i] = w @ v[:n]
        mag[i] = w @ np.abs(v[:n])
        big[i] = (np.abs(k[:n]) @ np.abs(q[i])).max() * scale
    return out, mag, big

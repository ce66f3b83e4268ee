"""Plain numpy restatement of the 8-bit cache (float64 where values are computed, exact bit tables for the codes), for
tests only: nothing here is fast and nothing is shared with the operators."""
from __future__ import annotations

import math

import numpy as np

BLOCK, TOP, E_MIN, E_MAX, NAN_CODE = 64, 448.0, -100, 120, 0x7F


def code_values() -> np.ndarray:
    """The 256 e4m3 values by code: sign, 4 exponent bits (bias 7), 3 fraction bits; 0x7f and 0xff are NaN."""
    out = np.empty(256)
    for c in range(256):
        e, f = (c >> 3) & 15, c & 7
        v = f / 8 * 2.0 ** -6 if e == 0 else (1 + f / 8) * 2.0 ** (e - 7)
        out[c] = math.nan if (c & 0x7F) == NAN_CODE else (-v if c & 0x80 else v)
    return out


_VALUES = code_values()
_POSITIVE = _VALUES[:NAN_CODE]                      # 0 .. 448, ascending


def encode(x: np.ndarray) -> np.ndarray:
    """The nearest code of each value (ties to the even code), values at most 448 in magnitude; non-finite -> NaN."""
    x = np.asarray(x, dtype=np.float64)
    a = np.abs(np.where(np.isfinite(x), x, 0.0))
    hi = np.clip(np.searchsorted(_POSITIVE, a), 0, NAN_CODE - 1)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - _POSITIVE[lo], _POSITIVE[hi] - a
    take_lo = (dl < dh) | ((dl == dh) & (lo % 2 == 0))
    c = np.where(take_lo, lo, hi) | np.where(np.signbit(x), 0x80, 0)
    return np.where(np.isfinite(x), c, NAN_CODE).astype(np.uint8)


def exponent(amax: float) -> int:
    """The smallest e in [-100, 120] with amax <= 448 * 2^e."""
    e = E_MIN
    while e < E_MAX and amax > math.ldexp(TOP, e):
        e += 1
    return e


def rotate(x: np.ndarray, table: np.ndarray, positions: np.ndarray, layout: str, inverse: bool = False) -> np.ndarray:
    """x [..., T, d] at positions [T] (or broadcastable), in x's precision with every product and sum rounded on its
    own; negative positions give zeros."""
    dt, half = x.dtype, table.shape[1] // 2
    rows = table[np.maximum(positions, 0)].astype(dt)
    c, s = rows[..., :half], rows[..., half:]
    s = -s if inverse else s
    y = x.copy()
    if layout == "half":
        a, b = x[..., :half], x[..., half:2 * half]
        y[..., :half], y[..., half:2 * half] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = a * c - b * s, b * c + a * s
    return np.where((positions >= 0)[..., None], y, np.zeros((), dt))


def append(codes: np.ndarray, exps: np.ndarray, new: np.ndarray, length: int) -> None:
    """One (batch, group): codes uint8 [C,d], exps int8 [NB], new [T,d]; row t goes to position length - T + t."""
    C, T = codes.shape[0], new.shape[0]
    start = length - T
    for blk in range(max(start, 0) // BLOCK, -(-min(length, C) // BLOCK)):
        p0 = blk * BLOCK
        lo, hi = max(p0, start), min(p0 + BLOCK, length, C)
        x = new[lo - start:hi - start].astype(np.float64)
        fin = np.abs(x[np.isfinite(x)])
        e = exponent(float(fin.max()) if fin.size else 0.0)
        if start > p0:
            e_old = int(exps[blk])
            e = max(e, e_old)
            codes[p0:lo] = encode(_VALUES[codes[p0:lo]] * 2.0 ** (e_old - e)) if e != e_old else codes[p0:lo]
        codes[lo:hi] = encode(x * 2.0 ** -e)
        exps[blk] = e


def values(codes: np.ndarray, exps: np.ndarray) -> np.ndarray:
    """codes uint8 [..., C, d], exps [..., NB] -> float64 values."""
    scale = np.repeat(np.exp2(exps.astype(np.float64)), BLOCK, axis=-1)[..., :codes.shape[-2]]
    return _VALUES[codes] * scale[..., None]


def sees(p: int, j: np.ndarray, window: int, sinks: int) -> np.ndarray:
    if window == 0:
        return j <= p
    return (j <= p) & ((j > p - window) | (j < sinks))


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, length: int, window: int, sinks: int, scale: float):
    """One (batch, group): q [h,T,d], k, v [C,d] values. Returns (out, sum of p |v|, largest sum of |q||k| * |scale|)
    in float64; a row that sees nothing is zero."""
    h, T, d = q.shape
    out, mass, mag = np.zeros((h, T, d)), np.zeros((h, T, d)), 0.0
    for t in range(T):
        p = length - T + t
        if p < 0:
            continue
        j = np.nonzero(sees(p, np.arange(length), window, sinks))[0]
        if j.size == 0:
            continue
        kk, vv = k[j], v[j]
        for i in range(h):
            s = kk @ q[i, t] * scale
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i, t], mass[i, t] = w @ vv, w @ np.abs(vv)
            mag = max(mag, float((np.abs(kk) @ np.abs(q[i, t])).max()) * abs(scale))
    return out, mass, mag

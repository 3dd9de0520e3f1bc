"""The 8-bit paged cache restated in numpy float64, straight from its definition.

Codes are e4m3 (sign, 4 exponent bits with bias 7, 3 mantissa bits; 0x7f / 0xff
are NaN, no infinities), one power-of-two scale per (layer, block, KV head) for
K and one for V; a stored value is code * scale.  Test infrastructure only."""

from __future__ import annotations

import numpy as np

MIN_EXP, MAX_EXP = -100, 119


def _code_values() -> np.ndarray:
    v = np.empty(256, dtype=np.float64)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        if e == 15 and m == 7:
            x = np.nan
        v[c] = -x if c >= 128 else x
    return v


VALUES = _code_values()
POSITIVE = VALUES[:127]  # ascending, codes 0 .. 126


def encode(x: np.ndarray) -> np.ndarray:
    """Nearest code of each value, ties to the even code, saturating; NaN -> 0x7f."""
    x = np.asarray(x, dtype=np.float64)
    a = np.minimum(np.abs(np.where(np.isnan(x), 0.0, x)), 448.0)
    hi = np.clip(np.searchsorted(POSITIVE, a), 1, 126)
    lo = hi - 1
    dl, dh = a - POSITIVE[lo], POSITIVE[hi] - a
    c = np.where(dl < dh, lo, np.where(dh < dl, hi, np.where(lo % 2 == 0, lo, hi)))
    c = np.where(np.signbit(x), c + 128, c)
    return np.where(np.isnan(x), 0x7F, c).astype(np.uint8)


def needed_scale(amax: float) -> float:
    """Smallest 2^k >= amax / 448, k in [MIN_EXP, MAX_EXP]."""
    k = MIN_EXP
    while k < MAX_EXP and amax > 448.0 * 2.0 ** k:
        k += 1
    return 2.0 ** k


def append(codes: np.ndarray, scales: np.ndarray, layer: int, table: np.ndarray, start: int, new: np.ndarray) -> None:
    """One row's append of ``new`` [Hkv, n, D] (float64) at ``start``, in place."""
    bs = codes.shape[3]
    end = start + new.shape[1]
    for j in range(start // bs, -(-end // bs)):
        p0, p1 = max(start, j * bs), min(end, (j + 1) * bs)
        blk, kept = int(table[j]), p0 - j * bs
        for h in range(codes.shape[2]):
            part = new[h, p0 - start:p1 - start]
            finite = np.abs(part[np.isfinite(part)])
            need = needed_scale(float(finite.max()) if finite.size else 0.0)
            old = float(scales[layer, blk, h])
            use = max(need, old) if kept else need
            page = codes[layer, blk, h]
            if kept and use > old:
                page[:kept] = encode(VALUES[page[:kept]] * (old / use))
            page[kept:p1 - j * bs] = encode(part / use)
            scales[layer, blk, h] = use


def read(codes: np.ndarray, scales: np.ndarray, layer: int, table: np.ndarray, n: int) -> np.ndarray:
    """One row's first ``n`` cached values, [Hkv, n, D] float64."""
    bs = codes.shape[3]
    ids = np.asarray(table[: -(-n // bs)], dtype=np.int64)
    x = VALUES[codes[layer][ids]] * scales[layer][ids].astype(np.float64)[:, :, None, None]
    h, d = codes.shape[2], codes.shape[4]
    return x.transpose(1, 0, 2, 3).reshape(h, -1, d)[:, :n]


def attention(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float | None = None):
    """Bottom-right causal attention of q [Hq, C, D] over k / v [Hkv, n, D].

    Returns (out [Hq, C, D], spread [Hq, C, D], reach [Hq, C], flat [Hq, C]): the
    result; the softmax-weighted mean of |v|, which bounds what a relative error
    of the weights can change; and, over the keys that a query sees, the
    largest sums of |q_d k_d| * scale and of max |q| |k_d| * scale, which bound
    the error of a score.  Queries that see no key give zeros."""
    hq, c, d = q.shape
    n, g = k.shape[1], hq // k.shape[0]
    scale = 1.0 / np.sqrt(d) if scale is None else scale
    out, spread, reach, flat = np.zeros((hq, c, d)), np.zeros((hq, c, d)), np.zeros((hq, c)), np.zeros((hq, c))
    if n == 0:
        return out, spread, reach, flat
    seen = np.arange(n)[None] <= n - c + np.arange(c)[:, None]
    for h in range(hq):
        z = np.where(seen, q[h] @ k[h // g].T * scale, -np.inf)
        top = z.max(axis=1, keepdims=True)
        p = np.exp(z - np.where(np.isfinite(top), top, 0.0))
        den = p.sum(axis=1, keepdims=True)
        p /= np.where(den > 0, den, 1.0)
        out[h], spread[h] = p @ v[h // g], p @ np.abs(v[h // g])
        reach[h] = np.where(seen, np.abs(q[h]) @ np.abs(k[h // g]).T * scale, 0.0).max(axis=1)
        flat[h] = np.where(seen, np.abs(k[h // g]).sum(axis=1)[None], 0.0).max(axis=1) * np.abs(q[h]).max(axis=1) * scale
    return out, spread, reach, flat

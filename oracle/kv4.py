"""Numpy restatement of the 4-bit KV cache (joule_moe.h, jl_kv4): the record's
quantiser in its own rules, the block layout by index arithmetic, and the
attention in 64 bits. Test infrastructure only."""
from __future__ import annotations

import numpy as np

BLOCK = 64


def quantise(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """rows [..., hd] -> codes 0..15 [..., hd] and fp16 scales [..., hd / 64].
    The rules of oracle/q4.py's record, with a scale of at most 65504 and NaN
    as zero; divisions in 64 bits, whose quotients fall on the same side of
    every step as the exact ones."""
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 64)
    a = np.abs(g)
    amax = np.maximum(np.where(np.isnan(a), 0.0, a).max(-1, keepdims=True), 1e-12)
    s = np.minimum(amax / 7.0, 65504.0).astype(np.float16)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = g / s.astype(np.float64)
    n = np.where(np.isnan(q), 0, np.clip(np.rint(np.nan_to_num(q, posinf=9, neginf=-9)), -8, 7)) + 8
    return n.astype(np.uint8).reshape(x.shape), s[..., 0]


def held(x: np.ndarray) -> np.ndarray:
    """The values that the cache holds of rows x, in 64 bits."""
    n, s = quantise(x)
    v = (n.astype(np.float64).reshape(*x.shape[:-1], -1, 64) - 8) * s.astype(np.float64)[..., None]
    return v.reshape(x.shape)


def byte_of(hd: int, is_v: bool, r: int, d: int) -> int:
    """Byte of value d of row r in a block (its nibble: d % 2, low first)."""
    ng, g, u = hd // 64, d // 64, d % 64 // 8
    if is_v:
        place = r // 8 * 8 + (0, 4, 1, 5, 2, 6, 3, 7)[r % 8]
        if r % 8 >= 4:
            u = (u + 4) % 8
        return 34 * hd + place * hd // 2 + 4 * (u * ng + g) + d % 8 // 2
    return r * hd // 2 + 4 * (u * ng + g) + d % 8 // 2


def scale_byte(hd: int, is_v: bool, r: int, g: int) -> int:
    return (66 if is_v else 32) * hd + 2 * (r * (hd // 64) + g)


def pack_block(k: np.ndarray, v: np.ndarray) -> np.ndarray:
    """uint8 [68 * hd] of rows k, v [n <= 64, hd]; rows past n are zero bytes."""
    n, hd = k.shape
    out = np.zeros(68 * hd, np.uint8)
    for is_v, x in ((False, k), (True, v)):
        codes, s = quantise(x)
        for r in range(n):
            for d in range(hd):
                out[byte_of(hd, is_v, r, d)] |= codes[r, d] << (4 * (d % 2))
            for g in range(hd // 64):
                b = scale_byte(hd, is_v, r, g)
                out[b:b + 2] = np.frombuffer(s[r, g].tobytes(), np.uint8)
    return out


def attention(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float) -> tuple[np.ndarray, np.ndarray, float]:
    """One sequence in 64 bits: q [T, H, hd] over cached values k, v [n, n_kv, hd];
    query i sees the first n - T + 1 + i rows. Returns out [T, H, hd], the
    largest |q| . |k| of each row (for error bounds) [T, H], and the largest |score|."""
    T, H, hd = q.shape
    n, kh = k.shape[:2]
    out, absdot, top = np.zeros((T, H, hd)), np.zeros((T, H)), 0.0
    for h in range(H):
        kk, vv = k[:, h // (H // kh)], v[:, h // (H // kh)]
        for i in range(T):
            m = n - T + 1 + i
            if m <= 0:
                continue
            s = scale * (kk[:m] @ q[i, h])
            absdot[i, h] = np.max(np.abs(kk[:m]) @ np.abs(q[i, h]))
            top = max(top, float(np.max(np.abs(s))))
            p = np.exp(s - s.max())
            out[i, h] = p @ vv[:m] / p.sum()
    return out, absdot, top

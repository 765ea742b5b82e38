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


def decode_step(model, x: np.ndarray, positions, cached):
    """The decode step of oracle/joule_oracle.c (jo_decode_step) with attention in
    64 bits over given cached values: cached(l, b) -> (k, v) [positions[b] + 1, n_kv,
    hd], this step's own row the last of them. Norms, RoPE and the MoE layers are the
    restatement's, the projections in 64 bits, rounded to fp32 where the step keeps
    fp32 rows. x [B, d] embedded inputs. Returns logits [B, V] (64 bits), the
    rows that the step appends (k, v [L][B, n_kv, hd] fp32), and the largest |score|."""
    import ctypes

    from oracle import restate
    lib, s, w = restate.lib(), model.shape, model.w
    lib.jo_rms_norm.argtypes = [ctypes.c_void_p] * 3 + [ctypes.c_int, ctypes.c_float]
    lib.jo_rope.argtypes = [ctypes.c_void_p] * 3 + [ctypes.c_int]
    lib.jo_sqrtf_fast.argtypes, lib.jo_sqrtf_fast.restype = [ctypes.c_float], ctypes.c_float
    f32 = lambda bits: (np.asarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32)  # noqa: E731

    def norm(rows, weight):
        rows = np.ascontiguousarray(rows, np.float32)
        out, weight = np.empty_like(rows), np.ascontiguousarray(weight)
        for i in range(rows.shape[0]):
            lib.jo_rms_norm(out[i].ctypes.data, rows[i].ctypes.data, weight.ctypes.data, rows.shape[1], s.eps)
        return out

    B, qn, kn = x.shape[0], s.H * s.hd, s.KH * s.hd
    h = np.array(x, np.float32)
    scale = 1.0 / float(np.float32(lib.jo_sqrtf_fast(float(s.hd))))
    ks, vs, top = [], [], 0.0
    for l in range(s.L):
        t = norm(h, w["norm1"][l])
        rows = []
        for name, bias, n in (("wq", "bq", qn), ("wk", "bk", kn), ("wv", "bv", kn)):
            r = t.astype(np.float64) @ f32(w[name][l]).astype(np.float64).T
            rows.append((r + (w[bias][l] if s.bias_qkv else 0.0)).astype(np.float32))
        q, k, v = rows
        if s.qk_norm_type == 2:
            q, k = norm(q, w["qn"][l]), norm(k, w["kn"][l])
        elif s.qk_norm_type == 1:
            q = norm(q.reshape(-1, s.hd), w["qn"][l]).reshape(B, qn)
            k = norm(k.reshape(-1, s.hd), w["kn"][l]).reshape(B, kn)
        q, k = np.ascontiguousarray(q), np.ascontiguousarray(k)
        for b in range(B):
            cs, sn = w["cos"][positions[b]], w["sin"][positions[b]]
            for r, heads in ((q[b], s.H), (k[b], s.KH)):
                for i in range(heads):
                    lib.jo_rope(r.ctypes.data + 4 * i * s.hd, cs.ctypes.data, sn.ctypes.data, s.hd)
        ks.append(k.reshape(B, s.KH, s.hd).copy())
        vs.append(v.reshape(B, s.KH, s.hd).copy())
        att = np.empty((B, qn))
        for b in range(B):
            kc, vc = cached(l, b)
            o, _, m = attention(q[b].reshape(1, s.H, s.hd).astype(np.float64), kc, vc, scale)
            att[b], top = o.reshape(qn), max(top, m)
        h = (h + att @ f32(w["wo"][l]).astype(np.float64).T).astype(np.float32)
        t = norm(h, w["norm2"][l])
        h = (h + restate.moe_layer(model.layers[l], t)[0]).astype(np.float32)
    return norm(h, w["final_norm"]).astype(np.float64) @ w["lm_head"].astype(np.float64).T, ks, vs, top

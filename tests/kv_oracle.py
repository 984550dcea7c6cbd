"""The quantized KV cache in plain numpy: the block formats' quantizers with the roundings that ggml's
reference ones make, what the codes stand for, and attention in 64 bits with the error that fp16
operands may cause (every rounding of an fp16 value is off by at most 2^-11 of it)."""
import numpy as np

Q4_0, Q8_0 = 2, 8
HALF = 2.0 ** -11          # fp16: half a step, relative


def f32(a):
    return np.asarray(a).astype(np.float32)


def quantize(x, t):
    """x f32 [..., D] -> (codes int8 [..., D] or uint8 [..., D / 2], scales fp16 [..., D / 32]). All
    arithmetic is numpy's f32, which rounds each step to nearest."""
    x = f32(x)
    b = x.reshape(x.shape[:-1] + (-1, 32))
    with np.errstate(all="ignore"):
        peak = np.take_along_axis(b, np.abs(b).argmax(-1)[..., None], -1)
        d = np.abs(peak) / np.float32(127) if t == Q8_0 else peak / np.float32(-8)
        inv = np.where(d != 0, np.float32(1) / d, np.float32(0))
        ok = np.isfinite(b).all(-1, keepdims=True)
        inv = np.where(ok & np.isfinite(inv), inv, np.float32(0))
        y = np.where(ok, b, np.float32(0)) * inv
        dh = np.where(ok, d, np.float32(np.nan)).astype(np.float16)[..., 0]
    if t == Q8_0:
        y64 = y.astype(np.float64)
        c = np.sign(y64) * np.floor(np.abs(y64) + 0.5)
        return c.astype(np.int8).reshape(x.shape), dh
    u = np.minimum(15, np.trunc(y + np.float32(8.5))).astype(np.uint8)
    return (u[..., :16] | (u[..., 16:] << 4)).reshape(x.shape[:-1] + (-1,)), dh


def values(codes, d, t):
    """What a cache stands for, f64."""
    d64 = d.astype(np.float64)[..., None]
    if t == Q8_0:
        c = codes.astype(np.float64).reshape(d.shape + (32,))
    else:
        u = codes.reshape(d.shape + (16,))
        c = np.concatenate([u & 15, u >> 4], -1).astype(np.float64) - 8
    with np.errstate(invalid="ignore"):
        v = c * d64
    return v.reshape(d.shape[:-1] + (-1,))


def held(codes, d, t):
    """The values attention takes: scales count as at most 515.5 (Q8_0) or 8188 (Q4_0), so that they stay
    inside fp16."""
    lim = np.float16(515.5 if t == Q8_0 else 8188)
    return values(codes, np.clip(d, -lim, lim), t)


def attention(q, k, v, mask, scale, softcap=0.0):
    """(dst, bound) of one sequence: q [H][T][D], k [HK][KV][D], v [HK][KV][DV] f64 values, mask [T][KV]
    f64 (-inf hides) or None. dst [T][H][DV] in 64 bits. bound: how far fp16 operands may take an
    output. Q and K rounded once each move a score by at most e = scale * sum|q||k| * (2 * HALF +
    HALF^2), a soft-cap by no more; P and the row sum then move by a factor within exp(+-2 e), P and V
    are rounded once each, and a P under fp16's normal range by at most 2^-25; f32 sums add the last
    2^-12 (64k terms at 2^-24, roots of which survive: the bound is loose here). The kernel that reads the cache
    as it is stored rounds V with its code's offset, d * (code + 128) or d * (code + 8), at most 255 d or
    15 d where a block's largest value is 127 d or 7 d at least (a largest negative code is 8 d): off by
    at most HALF * 15 / 7 of the largest magnitude in the block, instead of HALF of the value."""
    q, k, v = (np.asarray(a, dtype=np.float64) for a in (q, k, v))
    H, T, D = q.shape
    HK, KV, DV = v.shape
    out, tol = np.zeros((T, H, DV)), np.zeros((T, H, DV))
    # the largest magnitude of each block of 32 dims, times 15 / 7
    vmax = np.repeat(np.abs(v).reshape(HK, KV, DV // 32, 32).max(-1), 32, -1) * (15 / 7)
    for h in range(H):
        kh, vh = k[h * HK // H], v[h * HK // H]
        for t in range(T):
            m = np.zeros(KV) if mask is None else np.asarray(mask[t][:KV], dtype=np.float64)
            see = m != -np.inf
            if not see.any():
                continue
            ks, vs, vb = kh[see], vh[see], vmax[h * HK // H][see]
            x = ks @ q[h, t] * scale
            if softcap:
                x = softcap * np.tanh(x / softcap)
            x = x + m[see]
            p = np.exp(x - x.max())
            e = float((np.abs(ks) @ np.abs(q[h, t])).max()) * abs(scale) * (2 * HALF + HALF ** 2)
            size = p @ np.abs(vs) / p.sum()
            out[t, h] = p @ vs / p.sum()
            with np.errstate(over="ignore", invalid="ignore"):   # however the weights move, outputs stay among the values
                moved = np.minimum(np.where(size > 0, size * np.expm1(2 * e), np.inf), 2 * np.abs(vs).max(0))
            tol[t, h] = moved + size * (HALF + 2.0 ** -12) + (p @ vb / p.sum()) * HALF + see.sum() * 2.0 ** -25 * np.abs(vs).max()
    return out, tol

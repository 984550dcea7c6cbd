"""How far attention read directly from a cache in pages may be from 64 bits, a row and a 32-dim block of it at a time: as
kv_norm, without the roundings of Q and K that the direct forms do not make."""
import numpy as np

import kv_oracle as R
import pages_oracle as P

SIGMAS = 5.0
Q_HALVES, Q_F32, Q_F16 = 2.0 ** -22, 2.0 ** -27, 2.0 ** -35    # what F32 queries may lose of each value and of a row's largest; fp16 rows of theirs
STEPS = 8                                 # F32 roundings of a block's product, those inside the matrix unit among them


def mask_of(n_past, fresh, T, parents):
    m = np.full((T, n_past + fresh), -np.inf)
    for t, way in enumerate(P.ways(parents, fresh)):
        if way is not None:
            m[t, :n_past] = 0
            m[t, [n_past + u for u in way]] = 0
    return m


def attention(q, k, v, mask, scale, softcap=0.0, kd=None, vd=None, kt=P.F16, q_f16=False, half_out=False):
    """(dst [T][H][DV], sigma [T][H][DV / 32]) of one sequence: q [H][T][D], k [HK][KV][D], v [HK][KV][DV] f64 values, mask
    [T][KV] f64; kd, vd [HK][KV][dims / 32]: the block scales, None for an F16 cache (of type kt).

    Taken as independent and uniform (s off at most has the variance s^2 / 3). A score's error, e_j:
      Q                      F32, two halves: 2^-22 of each value and, the low half below fp16's normal range, 2^-25 of what a row in
                             [2^-2, 2^7) is times 2^8, over Q4_0 of 1/16 of it: 2^-21 / 2^6 of the row's largest. fp16: what falls
                             below 2^-24 where a row's largest value is brought down to 2^14, in 1/16 of it: 2^-21 / 2^14.
                             sqrt(sum (dq k)^2) scale
      its sum in F32         STEPS roundings of each block of 32 dims, 2^-24 of the largest that it holds: codes are multiplied as
                             unsigned ones, so 255 d sum |q| (Q4_0: 15 d); without codes sum |q k| of all dims. The matrix unit
                             lines products up by their operands' exponent fields, and a code u 2^-24 has the field of 2^-14, so
                             that it counts as 2^10 where it is u: 1024 d max |q| beside that
      the running sum, the product with scale log2(e), less the maximum: 2^-24 of |x| and of the largest |x|, 4 times
      a soft-cap             2e-7 of the cap; what comes before it arrives shrunk, never grown
      2^x                    2^-23 of the weight
    P:
      quantized V            P d rounded once (HALF of the term w v), the sum of the weights from P before that
      F16                    P rounded once, the sum that of the rounded ones: HALF of w (v - o)
      below fp16's normal range P is off by 2^-25, and P d by 2^-32 of the dims' largest d, a code of 255
    F32 sums, a 32-key step  2^-24 of 255 sum w d, or of sum w |v|, the largest that they hold.
    Through the weights e_j gives w e_j (v - o). The variance is the sum of all, sigma its root."""
    q, k, v = (np.asarray(a, dtype=np.float64) for a in (q, k, v))
    H, T, D = q.shape
    HK, KV, DV = v.shape
    nb, kb = DV // 32, D // 32
    out, sigma = np.zeros((T, H, DV)), np.zeros((T, H, nb))
    see = np.asarray(mask) != -np.inf
    for hk in range(HK):
        heads = np.arange(hk * H // HK, (hk + 1) * H // HK)
        qh, kh, vh = q[heads], k[hk], v[hk]                                   # [G][T][D]
        x = qh @ kh.T * scale
        amax = np.abs(qh).max(-1, keepdims=True)
        dq = Q_F16 * amax + 0 * qh if q_f16 else Q_F32 * amax + Q_HALVES * np.abs(qh)
        var = dq ** 2 @ (kh ** 2).T * scale ** 2 / 3
        if kd is None:
            var = var + STEPS * kb * 2.0 ** -48 / 3 * (np.abs(qh) @ np.abs(kh).T * scale) ** 2
        else:
            unit = 255.0 if kt == R.Q8_0 else 15.0
            qb = np.abs(qh).reshape(*qh.shape[:2], kb, 32)
            held = (unit * qb.sum(-1)) ** 2 + (1024 * qb.max(-1)) ** 2
            var = var + STEPS * 2.0 ** -48 / 3 * scale ** 2 * (held @ (np.abs(np.asarray(kd, dtype=np.float64)[hk]) ** 2).T)
        if softcap:
            x = softcap * np.tanh(x / softcap)
            var = var + (2e-7 * softcap) ** 2
        big = np.where(see, np.abs(x), 0).max(-1, keepdims=True)
        var = var + (kb + 8) * 2.0 ** -48 / 3 * (np.abs(x) ** 2 + big ** 2) + 2.0 ** -46 / 3
        x = np.where(see, x, -np.inf)
        top = x.max(-1, keepdims=True, initial=-np.inf)
        w = np.where(see, np.exp(x - np.where(top == -np.inf, 0, top)), 0.0)
        L = w.sum(-1, keepdims=True)
        inv = np.divide(1.0, L, out=np.zeros_like(L), where=L > 0)
        w = w * inv
        o = w @ vh                                                            # [G][T][DV]
        cut = lambda a: a.reshape(*a.shape[:-1], nb, 32)  # noqa: E731
        vb, ob = (cut(vh) ** 2).sum(-1), (cut(o) ** 2).sum(-1)

        def apart(a):   # sum_j a_j |v_j - o|^2
            return a @ vb - 2 * (cut(a @ vh) * cut(o)).sum(-1) + a.sum(-1, keepdims=True) * ob

        once = R.HALF ** 2 / 3
        e = apart(w ** 2 * var)
        if vd is None:
            e = e + apart(w ** 2 * once) + inv ** 2 * 2.0 ** -50 / 3 * apart(see.astype(float)[None] * np.ones_like(w))
            e = e + 32 * 2.0 ** -48 * (KV / 32 + 1) * ((w @ np.abs(cut(vh)).max(-1)) ** 2)
        else:
            d = np.abs(np.asarray(vd, dtype=np.float64)[hk])
            e = e + (w ** 2 * once) @ vb
            n = see.sum(-1)[None, :, None]
            e = e + 32 * 255 ** 2 * (2.0 ** -64 / 3 * n * (inv * d.max(0)) ** 2 + 2.0 ** -48 * (n / 32 + 1) * (w @ d) ** 2)
        if half_out:
            e = e + once * ob + 32 * 2.0 ** -50 / 3
        out[:, heads] = o.transpose(1, 0, 2)
        sigma[:, heads] = np.sqrt(np.maximum(e, 0)).transpose(1, 0, 2)
    return out, sigma


def errors(got, want, sigma):
    """(the largest error of a row's block over SIGMAS sigma, the root of all squared errors over that of all variances): the first at most 1, the
    second at most 1 but for chance, a few hundred rows' worth of it. NaN counts as infinite."""
    d = ((np.asarray(got, dtype=np.float64) - want).reshape(*sigma.shape, 32) ** 2).sum(-1)
    if np.isnan(d).any():
        return float("inf"), float("inf")
    with np.errstate(invalid="ignore", divide="ignore"):
        most = np.where(d == 0, 0.0, np.sqrt(d) / (SIGMAS * sigma)).max()
    return float(most), float(np.sqrt(d.sum() / max(float((sigma ** 2).sum()), 1e-300)))

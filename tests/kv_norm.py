"""How far attention over a quantized cache may be from 64 bits, a row and a 32-dim block of it at a time, as the root
of the sum of its roundings' squares. (kv_oracle.attention bounds every output for itself by the worst case, which
long rows never come near; this one notices a key that is missing.)"""
import numpy as np

import kv_oracle as R

SIGMAS = 5.0


def attention(q, k, v, mask, scale, softcap=0.0, vd=None, half_out=False):
    """(dst [T][H][DV], limit [T][H][DV / 32]) of one sequence: q [H][T][D], k [HK][KV][D], v [HK][KV][DV] f64 values,
    mask [T][KV] f64 or None; vd [HK][KV][DV / 32]: the scales of V's blocks (by default the largest |v| / 7, which the scale of
    a block whose largest value is 7 d or more does not pass).

    The roundings, taken as independent and uniform (half a step s off at most has the variance s^2 / 3), s = 2^-11 of
    the value for fp16:
      Q and K once each     a score is off by sigma_j = HALF sqrt(2 / 3) scale sqrt(sum q^2 k^2), values below fp16's
                            normal range by 2^-25 at most; the soft-cap's own 2e-7 of the cap on top
      P and V once each     (or their product once): HALF sqrt(2 / 3) of a key's term
    So key j's term w_j v_j, w its weight, is off by r_j = sqrt(sigma_j^2 + 2 HALF^2 / 3) of itself, and through the sum
    of the weights by as much of w_j o: sum_j (w_j r_j)^2 (|v_j|^2 + |o|^2) in all. Beside them, per key:
      P below fp16's normal range   2^-25 |v_j| (the largest P is 1 or more)
      V below it                    2^-25 w_j an element
      P d below it                  2^-32 of the dims' largest d, an unsigned code of 255 at most (where it is formed P is
                                    2^8 at most, d 2^7)
      F32 sums, a 32-key step       2^-24 of 255 sum w d, the largest that they hold
    The limit is SIGMAS times the root of the sum of all."""
    q, k, v = (np.asarray(a, dtype=np.float64) for a in (q, k, v))
    H, T, D = q.shape
    HK, KV, DV = v.shape
    nb = DV // 32
    out, limit = np.zeros((T, H, DV)), np.zeros((T, H, nb))
    m = np.zeros((T, KV)) if mask is None else np.asarray(mask, dtype=np.float64)[:T, :KV]
    see = m != -np.inf
    for hk in range(HK):
        heads = np.arange(hk * H // HK, (hk + 1) * H // HK)
        qh, kh, vh = q[heads], k[hk], v[hk]                                   # [G][T][D]
        x = qh @ kh.T * scale
        var = (qh ** 2 @ (kh ** 2).T) * scale ** 2 * (2 / 3) * R.HALF ** 2 + (kh ** 2).sum(-1) * (4 * 2.0 ** -50 / 3)
        if softcap:
            x = softcap * np.tanh(x / softcap)
            var = var + (2e-7 * softcap) ** 2
        x = x + m
        top = x.max(-1, keepdims=True)
        p = np.where(see, np.exp(x - np.where(top == -np.inf, 0, top)), 0.0)
        L = p.sum(-1, keepdims=True)
        w = np.divide(p, L, out=np.zeros_like(p), where=L > 0)
        o = w @ vh                                                            # [G][T][DV]
        vb = (vh.reshape(KV, nb, 32) ** 2).sum(-1)                            # [KV][nb]
        ob = (o.reshape(*o.shape[:2], nb, 32) ** 2).sum(-1)
        r2 = var + 2 * R.HALF ** 2 / 3
        e = (w ** 2 * r2) @ vb + (w ** 2 * r2).sum(-1, keepdims=True) * ob
        n = see.sum(-1)[None, :, None]
        inv = np.divide(1.0, L, out=np.zeros_like(L), where=L > 0)
        e += inv ** 2 * 2.0 ** -50 / 3 * (see.astype(float) @ vb)[None]
        e += 32 * 2.0 ** -50 / 3 * (w ** 2).sum(-1, keepdims=True)
        d = np.abs(vh).reshape(KV, nb, 32).max(2) / 7 if vd is None else np.abs(np.asarray(vd, dtype=np.float64)[hk])
        e += 32 * 255 ** 2 * (2.0 ** -64 / 3 * n * (inv * d.max(0)) ** 2 + 2.0 ** -48 * (n / 32 + 1) * (w @ d) ** 2)
        if half_out:
            e += R.HALF ** 2 / 3 * ob + 32 * 2.0 ** -50 / 3
        out[:, heads] = o.transpose(1, 0, 2)
        limit[:, heads] = SIGMAS * np.sqrt(e).transpose(1, 0, 2)
    return out, limit


def ratio(got, want, limit):
    """The largest error of a row's block over its limit (NaN counts as infinite)."""
    d = np.asarray(got, dtype=np.float64) - want
    d = np.sqrt((d.reshape(*limit.shape, 32) ** 2).sum(-1))
    with np.errstate(invalid="ignore", divide="ignore"):
        f = np.where(d == 0, 0.0, d / limit)
    return float(np.where(np.isnan(f), np.inf, f).max())

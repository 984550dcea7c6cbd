"""What pages_norm.errors lets pass and what not, with mistakes planted in plain numpy (CPU)."""
import numpy as np
import pytest

import kv_oracle as R
import pages_norm as N
import pages_oracle as P

CASES = [(P.F16, 2405, 4, 16, 64, 64), (R.Q8_0, 2405, 5, 8, 128, 128), (R.Q4_0, 5001, 1, 16, 128, 128), (R.Q4_0, 1000, 16, 4, 256, 256)]


def form(q, k, v, mask, scale, hide=(), twice=(), q_bits=True, t=P.F16):
    """The direct form's roundings in numpy: Q in two halves (q_bits False: one), P (F16) or P times the block's scale rounded to fp16."""
    qh = q.astype(np.float16).astype(np.float64)
    if q_bits:
        qh = qh + (q - qh).astype(np.float16)
    H, HK = q.shape[0], k.shape[0]
    out = np.zeros((q.shape[1], H, v.shape[2]))
    for h in range(H):
        x = qh[h] @ k[h * HK // H].T * scale + mask
        for at in hide:
            x[:, at:at + 32] = -np.inf
        p = np.exp(x - x.max(-1, keepdims=True))
        for at in twice:
            p[:, at:at + 32] *= 2
        r = p.astype(np.float16).astype(np.float64)
        out[:, h] = r @ v[h * HK // H] / (r if t == P.F16 else p).sum(-1, keepdims=True)
    return out


@pytest.mark.parametrize("t,KV,T,H,D,DV", CASES)
def test_notices(t, KV, T, H, D, DV):
    rng = np.random.default_rng(KV + D)
    HK = max(1, H // 4)
    pls = [P.planes(rng.standard_normal((KV, HK, d)).astype(np.float32), t) for d in (D, DV)]
    k, v = (P.cache_values(pl, t).transpose(1, 0, 2) for pl in pls)
    kd, vd = (None if t == P.F16 else pl[1].view(np.float16).astype(np.float64).transpose(1, 0, 2) for pl in pls)
    q, scale = 3 * rng.standard_normal((H, T, D)).astype(np.float32).astype(np.float64), D ** -0.5
    mask = N.mask_of(KV - T, T, T, None)
    want, sigma = N.attention(q, k, v, mask, scale, 0.0, kd, vd, t)
    most, whole = N.errors(form(q, k, v, mask, scale, t=t), want, sigma)
    assert most <= 1 and whole <= 1.1
    for at in (0, 32 * (KV // 64), (KV - T) // 32 * 32 - 32):       # the first tile, one in the middle, one before the last
        assert N.errors(form(q, k, v, mask, scale, hide=[at], t=t), want, sigma)[0] > 1
        assert N.errors(form(q, k, v, mask, scale, twice=[at], t=t), want, sigma)[0] > 1
    assert N.errors(form(q, k, v, mask, scale, q_bits=False, t=t), want, sigma)[1] > 1.1
    assert N.errors(np.full_like(want, np.nan), want, sigma) == (float("inf"), float("inf"))

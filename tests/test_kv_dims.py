"""Attention over a quantized cache at every pair of head dims it takes, under every form."""
import numpy as np
import pytest

import kv_norm
import kv_oracle as R
from test_kv_gpu import MIXES, cpu, form, gpu, mx  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", range(32, 257, 32))
def test_every_pair(mx, form, D):
    """All types, a partial last tile, two keys hidden, negative scales (a Q4_0 block's have either sign)."""
    H, HK, T, KV = 6, 2, 6, 75
    rng = np.random.default_rng(D)
    m = np.zeros((T, 76), np.float16)
    m[:, [5, 70]] = -np.inf
    for i, DV in enumerate(range(32, 257, 32)):
        kt, vt = MIXES[(i + D // 32) % 4]
        q = rng.standard_normal((H, T, D)).astype(np.float32)
        kq, kd = R.quantize(rng.standard_normal((KV, HK, D)), kt)
        vq, vd = R.quantize(rng.standard_normal((KV, HK, DV)), vt)
        kn, vn = (R.values(*c).transpose(1, 0, 2) for c in ((kq, kd, kt), (vq, vd, vt)))
        kc, vc = (mx.KvCache(t, gpu(c), gpu(d)).permute(1, 0, 2) for t, c, d in ((kt, kq, kd), (vt, vq, vd)))
        got = cpu(mx.flash_attn_q(gpu(q), kc, vc, gpu(m), D ** -0.5))
        want, limit = kv_norm.attention(q, kn, vn, m, D ** -0.5, vd=vd.transpose(1, 0, 2))
        assert kv_norm.ratio(got, want, limit) <= 1, (DV, kt, vt, kv_norm.ratio(got, want, limit))

"""Attention over a quantized cache with queries far below fp16's range, zeros among their values: all keys weigh
nearly the same, and nothing is infinite or NaN on the way."""
import numpy as np
import pytest

import kv_norm
import kv_oracle as R
from test_kv_gpu import MIXES, attn_case, cpu, form, gpu, ids, mx  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("types", MIXES, ids=ids)
@pytest.mark.parametrize("T,D,DV", [(1, 128, 128), (9, 96, 64), (20, 64, 64)])
def test_small_queries(mx, form, types, T, D, DV):
    """Row by row from 2^-7 down to F32's smallest; rows of zeros and rows with one value that is not zero."""
    H, HK, KV = 8, 2, 90
    q, kn, vn, kc, vc = attn_case(mx, *types, 1, T, H, HK, KV, D, DV)
    rng = np.random.default_rng(T)
    top = np.float64(2.0) ** np.linspace(-7, -148, H * T).reshape(H, T, 1)
    q = (rng.uniform(0.5, 1.0, q.shape[1:]) * rng.choice([-1, 0, 1], q.shape[1:]) * top).astype(np.float32)
    q[0, 0] = 0
    q[1, 0] = 0
    q[1, 0, D - 1] = np.float32(1e-45)
    q[2, 0] = 0
    q[2, 0, 3] = np.float32(-3e-39)
    m = np.where(np.arange(96)[None] > KV - T + np.arange(T)[:, None], -np.inf, 0.0).astype(np.float16)
    for scale in (D ** -0.5, 1.0):
        got = cpu(mx.flash_attn_q(gpu(q), kc[0], vc[0], gpu(m), scale))
        assert np.isfinite(got).all()
        want, limit = kv_norm.attention(q, kn[0], vn[0], m.astype(np.float64), scale)
        assert kv_norm.ratio(got, want, limit) <= 1

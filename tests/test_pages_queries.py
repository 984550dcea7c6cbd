"""Queries of any size over a cache in pages: what the direct forms keep of them, seen in scores of a thousand that nearly cancel."""
import numpy as np
import pytest

import pages_norm as N
import pages_oracle as P
from test_pages_gpu import ATTENDED, F16, NAME, cache_of, cpu, gpu, i32, mx, tables  # noqa: F401

pytestmark = pytest.mark.gpu

SPREAD = 1000.0     # a query of these keys' size at random would have scores of this spread
SIZES = [("F32", s) for s in (1e-20, 0.007, 0.02, 1.0, 40.0, 1e4, 1e20)] + [("F16", s) for s in (1e-5, 0.002, 0.02, 1.0, 100.0, 1e4)]


@pytest.mark.parametrize("kind,size", SIZES, ids=lambda v: v if isinstance(v, str) else "%g" % v)
@pytest.mark.parametrize("D,DV", [(64, 64), (128, 128), (192, 128), (256, 256)])
@pytest.mark.parametrize("kt,vt", ATTENDED, ids=lambda t: NAME[t])
def test_queries_keep_their_values(mx, monkeypatch, kt, vt, D, DV, kind, size):  # noqa: F811
    """32 keys, and for each head a query whose scores with them are within a few of each other, although query and keys are long: an error of the query
    moves every score by SPREAD times as much of itself."""
    monkeypatch.setenv("MI355X_FA_Q_DIRECT", "1")
    HK, KV, page = 64, 32, 32
    rng = np.random.default_rng(D)
    table, pages = tables(rng, [KV - 1], [1], page)
    at = [P.row(table[0], page, j) for j in range(KV)]
    (kc, kp), (vc, vp) = cache_of(mx, kt, pages * page, HK, D, rng), cache_of(mx, vt, pages * page, HK, DV, rng)
    k, v = (P.cache_values([p[at] for p in pl], t).transpose(1, 0, 2) for pl, t in ((kp, kt), (vp, vt)))
    scale = float(np.float32(SPREAD / (size * D ** 0.5)))
    q = rng.standard_normal((HK, D)) * size
    for h in range(HK):      # off the keys' span, then back by what gives the scores
        q[h] += k[h].T @ np.linalg.solve(k[h] @ k[h].T, 1.5 * rng.standard_normal(KV) / scale - k[h] @ q[h])
    q = q.astype(np.float32 if kind == "F32" else np.float16)
    step = mx.KvStep(i32(table), i32([KV - 1]), 1, page)
    got = cpu(mx.flash_attn_paged(gpu(q[None, :, None]), kc, vc, step, scale))[0]
    kd, vd = ((None if t == F16 else pl[1][at].view(np.float16).astype(np.float64).transpose(1, 0, 2)) for pl, t in ((kp, kt), (vp, vt)))
    want, sigma = N.attention(q[:, None].astype(np.float64), k, v, np.zeros((1, KV)), scale, 0.0, kd, vd, kt, kind == "F16")
    most, whole = N.errors(got, want, sigma)
    assert most <= 1 and whole <= 1.1, (most, whole)

"""Attention over a quantized cache whose V scales lie far apart, between the 32-dim blocks of a key and between keys:
every block of dims is as good as its own values allow, in every form."""
import numpy as np
import pytest

import kv_norm
import kv_oracle as R
from test_kv_gpu import cpu, form, gpu, ids, mx  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu

Q4_0, Q8_0 = R.Q4_0, R.Q8_0
H, HK, KV = 8, 2, 400


def run(mx, vt, D, DV, scales, mask, T):
    """V of N(0, 1) values times scales [KV][DV / 32] (of the blocks' largest values), against 64 bits."""
    rng = np.random.default_rng(DV + T)
    q = rng.standard_normal((H, T, D)).astype(np.float32)
    kq, kd = R.quantize(rng.standard_normal((KV, HK, D)), Q8_0)
    x = rng.standard_normal((KV, HK, DV // 32, 32))
    x *= (scales[:, None] / np.abs(x).max(-1))[..., None]
    vq, vd = R.quantize(x.reshape(KV, HK, DV), vt)
    kn, vn = (R.values(*c).transpose(1, 0, 2) for c in ((kq, kd, Q8_0), (vq, vd, vt)))
    kc, vc = (mx.KvCache(t, gpu(c), gpu(d)).permute(1, 0, 2) for t, c, d in ((Q8_0, kq, kd), (vt, vq, vd)))
    want, limit = kv_norm.attention(q, kn, vn, mask.astype(np.float64), D ** -0.5, vd=vd.transpose(1, 0, 2))
    for ns in (0, 1, 3):
        got = cpu(mx.flash_attn_q(gpu(q), kc, vc, gpu(mask), D ** -0.5, nsplit=ns))
        assert kv_norm.ratio(got, want, limit) <= 1, (ns, kv_norm.ratio(got, want, limit))


@pytest.mark.parametrize("vt", [Q8_0, Q4_0], ids=ids)
@pytest.mark.parametrize("DV", [64, 128, 256])
@pytest.mark.parametrize("T", [1, 9])
@pytest.mark.parametrize("ratio", [1e2, 1e4, 1e6])
def test_blocks_of_a_key_apart(mx, form, vt, DV, T, ratio):
    """Blocks of dims whose values are `ratio` apart, the small and the large ones in turn."""
    scales = np.ones((KV, DV // 32)) * 8000.0
    scales[:, 1::2] /= ratio
    mask = np.zeros((T, KV), np.float16)
    run(mx, vt, 64 if DV < 256 else 256, DV, scales, mask, T)


@pytest.mark.parametrize("vt", [Q8_0, Q4_0], ids=ids)
@pytest.mark.parametrize("DV", [64, 128])
@pytest.mark.parametrize("T", [1, 9])
@pytest.mark.parametrize("ratio", [1e4, 1e6])
def test_keys_apart(mx, form, vt, DV, T, ratio):
    """Some keys' values are `ratio` times the others'. They are visible, but their weight is nothing (a bias of -60),
    so outputs are the others', to their accuracy."""
    scales = np.full((KV, DV // 32), 8000.0 / ratio)
    mask = np.zeros((T, KV), np.float16)
    for j in (3, 40, 41, 200, 399):
        scales[j] = 8000.0
        mask[:, j] = -60.0
    run(mx, vt, 64, DV, scales, mask, T)

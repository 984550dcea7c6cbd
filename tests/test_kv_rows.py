"""Attention over a quantized cache row by row: close enough to 64 bits that one key more or less would show, and (on the
CPU) that it would."""
import numpy as np
import pytest

import kv_norm
import kv_oracle as R
from test_kv_gpu import MIXES, causal, cpu, form, gpu, ids, mx  # noqa: F401  (fixtures)

LENGTHS = [(1, 1), (1, 2), (1, 33), (1, 777), (3, 64), (7, 1000), (16, 129), (33, 500), (70, 389), (1, 2000), (1, 3000), (2, 8191)]
H, HK, D = 8, 2, 128


def case(types, T, KV, S=1, D=D, DV=D):
    rng = np.random.default_rng(1000 * T + KV + D)
    q = rng.standard_normal((S, H, T, D)).astype(np.float32)
    kq, kd = R.quantize(rng.standard_normal((S, KV, HK, D)), types[0])
    x = rng.standard_normal((S, KV, HK, DV))
    x[:, [0, -1]] *= 4          # the ends of a long row stand out
    vq, vd = R.quantize(x, types[1])
    vals = [R.values(*c).transpose(0, 2, 1, 3) for c in ((kq, kd, types[0]), (vq, vd, types[1]))]
    return q, vals[0], vals[1], vd.transpose(0, 2, 1, 3), ((types[0], kq, kd), (types[1], vq, vd))


@pytest.mark.gpu
@pytest.mark.parametrize("types", MIXES, ids=ids)
@pytest.mark.parametrize("T,KV", LENGTHS)
def test_rows(mx, form, types, T, KV):
    """Causal, GQA of four, whole and split."""
    q, k, v, vd, planes = case(types, T, KV)
    kc, vc = (mx.KvCache(t, gpu(c), gpu(d)).permute(0, 2, 1, 3) for t, c, d in planes)
    m = causal(T, KV)
    want, limit = kv_norm.attention(q[0], k[0], v[0], m[0], D ** -0.5, vd=vd[0])
    for ns in (0, 1, 3):
        got = cpu(mx.flash_attn_q(gpu(q), kc, vc, gpu(m), D ** -0.5, nsplit=ns))[0]
        assert kv_norm.ratio(got, want, limit) <= 1, (ns, kv_norm.ratio(got, want, limit))


@pytest.mark.gpu
@pytest.mark.parametrize("types", MIXES, ids=ids)
@pytest.mark.parametrize("D,DV", [(32, 32), (64, 64), (96, 96), (128, 64), (192, 128), (256, 256), (160, 96)])
@pytest.mark.parametrize("T,half", [(1, True), (12, False)])
def test_rows_of_other_head_dims(mx, form, types, D, DV, T, half):
    """Three sequences, fp16 queries and outputs, a soft-cap."""
    import torch
    S, KV, cap = 3, 301, 20.0
    q, k, v, vd, planes = case(types, T, KV, S, D, DV)
    if half:
        q = q.astype(np.float16)
    kc, vc = (mx.KvCache(t, gpu(c), gpu(d)).permute(0, 2, 1, 3) for t, c, d in planes)
    m = causal(T, KV, [301, 40, 160])
    out = torch.empty(S, T, H, DV, dtype=torch.float16 if half else torch.float32, device="cuda")
    got = cpu(mx.flash_attn_q(gpu(q), kc, vc, gpu(m), D ** -0.5, softcap=cap, out=out))
    for s in range(S):
        want, limit = kv_norm.attention(q[s].astype(np.float64), k[s], v[s], m[s], D ** -0.5, cap, vd[s], half_out=half)
        assert kv_norm.ratio(got[s], want, limit) <= 1, (s, kv_norm.ratio(got[s], want, limit))


def fp16_attention(q, k, v, m, scale):
    """The same with Q, K, P and V rounded to fp16."""
    q, k, v = (a.astype(np.float16).astype(np.float64) for a in (q * scale, k, v))
    x = np.repeat(k, H // HK, 0) @ q.transpose(0, 2, 1)                       # [H][KV][T]
    x = x.transpose(0, 2, 1) + m[None]
    p = np.exp(x - x.max(-1, keepdims=True)).astype(np.float16).astype(np.float64)
    return (p @ np.repeat(v, H // HK, 0) / p.sum(-1, keepdims=True)).transpose(1, 0, 2)


@pytest.mark.parametrize("types", MIXES, ids=ids)
@pytest.mark.parametrize("T,KV", LENGTHS)
def test_what_a_row_notices(types, T, KV):
    """Operands of fp16 pass; a result without the last key, with the first one twice, without a tile of 32 keys, or with
    one query seeing a key too many does not."""
    q, k, v, vd, _ = case(types, T, KV)
    q, k, v, m = q[0].astype(np.float64), k[0], v[0], causal(T, KV)[0][:, :KV].astype(np.float64)
    want, limit = kv_norm.attention(q, k, v, m, D ** -0.5, vd=vd[0])
    old, _ = R.attention(q[:, -1:], k, v, m[-1:], D ** -0.5)
    assert np.abs(old - want[-1:]).max() < 1e-12
    assert kv_norm.ratio(fp16_attention(q, k, v, m, D ** -0.5), want, limit) <= 1

    def wrong(mask, kk=k, vv=v):
        return kv_norm.ratio(kv_norm.attention(q, kk, vv, mask, D ** -0.5)[0], want, limit)
    less = m.copy()
    less[:, -1] = -np.inf
    assert wrong(less) > 1
    if KV > 1:
        twice = (np.concatenate([a, a[:, :1]], 1) for a in (k, v))
        assert wrong(np.concatenate([m, m[:, :1]], 1), *twice) > 1
    if KV > 64:
        hole = m.copy()
        hole[:, 32:64] = -np.inf
        assert wrong(hole) > 1
    if T > 1:
        more = m.copy()
        more[0, KV - T + 1] = 0
        assert wrong(more) > 1

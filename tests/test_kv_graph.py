"""FLASH_ATTN_EXT nodes over a quantized cache through the backend: what is claimed, the CPU form and the
device form, on ggml blocks in the strided views that a graph holds (a slice of a longer cache)."""
import json
import os
import subprocess
import sys

import numpy as np
import pytest

import ggml_mi355x as mx
import kv_oracle as R

HERE = os.path.dirname(os.path.abspath(__file__))
MIXES = [(mx.Q8_0, mx.Q8_0), (mx.Q4_0, mx.Q4_0), (mx.Q8_0, mx.Q4_0), (mx.Q4_0, mx.Q8_0)]

PROBE = """
import json, sys
sys.path[:0] = json.loads(sys.argv[1])
import ggml_mi355x as mx
def fa(kt, vt, D=128, DV=128, T=64, KV=2048, q=mx.F32, max_bias=0.0, knb=None):
    g = mx.Graph(alloc=False)
    kv = g.new_tensor(kt, [D, KV, 2, 1]), g.new_tensor(vt, [DV, KV, 2, 1])
    if knb:
        kv[0].nb[1] = knb
    return mx.supports_op(g.flash_attn_ext(g.new_tensor(q, [D, T, 8, 1]), *kv, g.new_tensor(mx.F16, [KV, T]), 1.0, max_bias))
print(json.dumps([fa(mx.Q8_0, mx.Q8_0), fa(mx.Q4_0, mx.Q4_0), fa(mx.Q8_0, mx.Q4_0), fa(mx.Q4_0, mx.Q8_0), fa(mx.Q8_0, mx.Q8_0, 192, 96),
                  fa(mx.F16, mx.F16), fa(mx.F16, mx.Q8_0), fa(mx.Q8_0, mx.F16), fa(mx.Q4_K, mx.Q4_K, 256, 256), fa(mx.Q8_0, mx.Q8_0, 288, 288),
                  fa(mx.Q8_0, mx.Q8_0, T=1), fa(mx.Q8_0, mx.Q8_0, KV=512), fa(mx.Q8_0, mx.Q8_0, q=mx.F16), fa(mx.Q8_0, mx.Q8_0, max_bias=1.0),
                  fa(mx.Q8_0, mx.Q8_0, knb=150)]))
"""


@pytest.mark.parametrize("knob,cache", [(None, False), ("1", True), ("0", False)])
def test_placement(knob, cache):
    """Claimed where FLASH_ATTN_QUANT is set, under the rules of an F16 cache; never one quantized side alone,
    another type, a head dim past 256 or rows that are not whole blocks apart."""
    e = {k: v for k, v in os.environ.items() if not k.startswith(("MI355X_", "ROCKET_"))}
    if knob is not None:
        e["MI355X_FLASH_ATTN_QUANT"] = knob
    r = subprocess.run([sys.executable, "-c", PROBE, json.dumps([os.path.dirname(mx.__file__), HERE])], env=e, capture_output=True,
                       text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    assert json.loads(r.stdout.strip().splitlines()[-1]) == [cache] * 5 + [True] + [False] * 9


def blocks(codes, d):
    """ggml blocks: the fp16 scale, then the block's codes."""
    c = codes.reshape(d.shape + (-1,)).view(np.uint8)
    return np.ascontiguousarray(np.concatenate([d[..., None].view(np.uint8), c], -1)).reshape(-1)


def graph(kt, vt, D, DV, T, H, HK, KV, n_ctx, softcap=0.0, seed=0, shared=False):
    rng = np.random.default_rng(seed + D + T + KV)
    g = mx.Graph()
    qv = rng.standard_normal((T, H, D)).astype(np.float32)
    qb = g.new_tensor(mx.F32, [D, H, T], "q_proj")
    g.set(qb, qv)
    q = g.permute_view(qb, [D, T, H, 1], [4, 4 * D * H, 4 * D, 4 * D * H * T])
    views, vals = [], []
    for t, w, name in ((kt, D, "cache_k_l0"), (vt, DV, "cache_v_l0")):
        if shared and views:      # V as the first dims of K's rows
            t, w, b = kt, DV, views[0][1]
            codes, d = views[0][2], views[0][3]
            row = D
        else:
            codes, d = R.quantize(rng.standard_normal((n_ctx, HK, w)), t)
            b = g.new_tensor(t, [w, HK, n_ctx], name)
            g.set(b, blocks(codes, d))
            row = w
        bb = 34 if t == mx.Q8_0 else 18
        hb = bb * row // 32
        views.append((g.permute_view(b, [w, KV, HK, 1], [bb, hb * HK, hb, hb * HK * n_ctx]), b, codes, d))
        vals.append(R.values(codes[:KV], d[:KV], t).transpose(1, 0, 2)[..., :w])
    m16 = np.where(np.arange(KV)[None, :] > KV - T + np.arange(T)[:, None], -np.inf, 0.0).astype(np.float16)
    m16[T // 2] = -np.inf
    m = g.new_tensor(mx.F16, [KV, T])
    g.set(m, m16)
    scale = float(np.float32(D ** -0.5))
    o = g.flash_attn_ext(q, views[0][0], views[1][0], m, scale, softcap=softcap)
    want, tol = R.attention(qv.transpose(1, 0, 2).astype(np.float64), *vals, m16.astype(np.float64), scale, softcap)
    return g, o, want, tol


CASES = [(128, 128, 16, 8, 2, 160, 256, 0.0), (64, 64, 33, 4, 4, 96, 96, 30.0), (192, 128, 17, 4, 1, 128, 200, 0.0)]


@pytest.mark.parametrize("types", MIXES)
@pytest.mark.parametrize("case", CASES)
def test_cpu_form(types, case):
    """What computes the node when the device does not: 64-bit arithmetic on the decoded blocks, rounded to F32
    once (2^-24, and the softmax's and soft-cap's own double roundings far below it)."""
    D, DV, T, H, HK, KV, n_ctx, cap = case
    be = mx.Backend()
    g, o, want, _ = graph(*types, D, DV, T, H, HK, KV, n_ctx, cap)
    be.inject_faults("fa", 1)
    assert be.compute([o]) == mx.STATUS_SUCCESS and be.cpu_fallbacks() == 1
    got = g.get(o, np.float32, (T, H, DV))
    assert (np.abs(got - want) <= 2.0 ** -23 * np.abs(want) + 1e-12).all()
    assert (got[T // 2] == 0).all()
    be.free()


@pytest.mark.gpu
@pytest.mark.parametrize("types", MIXES)
@pytest.mark.parametrize("case", CASES + [(128, 128, 512, 8, 2, 1100, 1200, 0.0), (128, 128, 300, 32, 8, 1056, 1100, 20.0)])
def test_device_form(torch_cuda, types, case):
    """On the device, twice over one backend (buffers of other sizes between), no fallback."""
    D, DV, T, H, HK, KV, n_ctx, cap = case
    be = mx.Backend()
    for seed in (0, 1):
        g, o, want, tol = graph(*types, D, DV, T, H, HK, KV, n_ctx + seed, cap, seed)
        assert be.compute([o]) == mx.STATUS_SUCCESS and be.cpu_fallbacks() == 0 and be.route_ops("fa") == 1 + seed
        got = g.get(o, np.float32, (T, H, DV))
        assert (np.abs(got - want) <= tol).all() and (got[T // 2] == 0).all()
    be.free()


@pytest.mark.gpu
def test_v_inside_k(torch_cuda):
    """V a view of the first dims of K's rows: one upload, one packing."""
    be = mx.Backend()
    g, o, want, tol = graph(mx.Q8_0, mx.Q8_0, 192, 128, 16, 8, 1, 140, 150, shared=True)
    assert be.compute([o]) == mx.STATUS_SUCCESS and be.cpu_fallbacks() == 0
    assert (np.abs(g.get(o, np.float32, (16, 8, 128)) - want) <= tol).all()
    be.free()


def test_one_quantized_side_is_computed_on_the_cpu():
    """A node that nothing claims, handed in all the same."""
    be = mx.Backend()
    g = mx.Graph()
    rng = np.random.default_rng(3)
    q, k, v = rng.standard_normal((2, 16, 64)).astype(np.float32), rng.standard_normal((1, 40, 64)), rng.standard_normal((1, 40, 64))
    kq, kd = R.quantize(k, mx.Q8_0)
    tq, tk, tv = g.new_tensor(mx.F32, [64, 16, 2]), g.new_tensor(mx.Q8_0, [64, 40, 1]), g.new_tensor(mx.F16, [64, 40, 1])
    g.set(tq, q), g.set(tk, blocks(kq, kd)), g.set(tv, v.astype(np.float16))
    o = g.flash_attn_ext(tq, tk, tv, None, 0.125)
    be.inject_faults("fa", 1)
    assert be.compute([o]) == mx.STATUS_SUCCESS and be.cpu_fallbacks() == 1
    want, _ = R.attention(q.astype(np.float64), R.values(kq, kd, mx.Q8_0), v.astype(np.float16).astype(np.float64), None, 0.125)
    assert (np.abs(g.get(o, np.float32, (16, 2, 64)) - want) <= 2.0 ** -23 * np.abs(want) + 1e-12).all()
    be.free()

"""What SET_ROWS, GET_ROWS and FLASH_ATTN_EXT of a quantized cache refuse, before touching the device (CPU)."""
import ctypes

import pytest
import torch

import ggml_mi355x as mx

FAKE = 1 << 20      # aligned, never dereferenced on these paths


def rows(**kw):
    a = dict(type=mx.Q8_0, q_dev=FAKE, d_dev=FAKE, n_rows=16, nb1=512, nb2=128, H=4, D=128, x_type=mx.F32, x_dev=FAKE, x_nb1=512, x_nb2=128)
    a.update(kw)
    return mx.KvRows(**a)


ROW_REFUSALS = [dict(type=mx.Q4_K), dict(type=mx.F32), dict(q_dev=None), dict(q_dev=FAKE + 8), dict(d_dev=None), dict(d_dev=FAKE + 2),
                dict(nb1=500), dict(nb2=16), dict(nb1=-512), dict(nb2=-128), dict(H=0), dict(D=0), dict(D=48), dict(D=1 << 40),
                dict(x_type=mx.BF16), dict(x_dev=None), dict(x_dev=FAKE + 4), dict(x_nb1=516), dict(x_nb2=-8), dict(n_rows=-1)]


@pytest.mark.parametrize("fn", ["mi355x_set_rows", "mi355x_get_rows"])
@pytest.mark.parametrize("bad", ROW_REFUSALS, ids=lambda b: "-".join(f"{k}={v}" for k, v in b.items()))
def test_rows_refusals(fn, bad):
    f = getattr(mx.lib(), fn)
    both = (mx.KvRows * 2)(rows(), rows(**bad))
    assert f(both, 2, FAKE, mx.I64, 3, None, None) == mx.E_ARG


@pytest.mark.parametrize("fn", ["mi355x_set_rows", "mi355x_get_rows"])
def test_rows_of_more_blocks_than_a_launch_counts(fn):
    two = (mx.KvRows * 2)(*[rows(H=32, D=1024, nb1=1 << 15, nb2=1024, x_nb1=1 << 15, x_nb2=1024)] * 2)
    assert getattr(mx.lib(), fn)(two, 2, FAKE, mx.I64, (1 << 19) + 1, None, None) == mx.E_ARG
    one = (mx.KvRows * 1)(rows(H=1 << 15, D=16416, nb1=1 << 30, nb2=16416, x_nb1=1 << 30, x_nb2=16416))
    assert getattr(mx.lib(), fn)(one, 1, FAKE, mx.I64, 1, None, None) == mx.E_ARG


@pytest.mark.parametrize("fn", ["mi355x_set_rows", "mi355x_get_rows"])
def test_rows_call_refusals(fn):
    f = getattr(mx.lib(), fn)
    one = (mx.KvRows * 1)(rows())
    five = (mx.KvRows * 5)(*[rows()] * 5)
    assert f(None, 1, FAKE, mx.I64, 3, None, None) == mx.E_ARG
    assert f(one, 0, FAKE, mx.I64, 3, None, None) == mx.E_ARG
    assert f(five, 5, FAKE, mx.I64, 3, None, None) == mx.E_ARG
    assert f(one, 1, FAKE, mx.I64, -1, None, None) == mx.E_ARG
    assert f(one, 1, FAKE, mx.I64, 1 << 31, None, None) == mx.E_ARG
    assert f(one, 1, FAKE, mx.F16, 3, None, None) == mx.E_ARG
    assert f(one, 1, FAKE + 4, mx.I64, 3, None, None) == mx.E_ARG
    assert f(one, 1, FAKE, mx.I32, 3, FAKE + 2, None) == mx.E_ARG
    assert f(one, 1, None, mx.I32, 17, None, None) == mx.E_ARG          # no indices: more rows than the cache has
    assert f(one, 1, FAKE, mx.I64, 0, None, None) == mx.OK
    empty = (mx.KvRows * 1)(rows(q_dev=None, d_dev=None, x_dev=None))
    assert f(empty, 1, None, mx.I32, 0, None, None) == mx.OK


def view(**kw):
    a = dict(type=mx.Q8_0, q_dev=FAKE, d_dev=FAKE, nb1=512, nb2=128, nb3=0)
    a.update(kw)
    return mx.KvView(**a)


def fa(k=None, v=None, **kw):
    a = dict(q_dev=FAKE, q_nb1=128, q_nb2=1024, q_nb3=0, k=view(**(k or {})), v=view(**(v or {})), mask_dev=FAKE, mask_nb1=64, mask_nb3=0,
             dst_dev=FAKE, dst_nb1=128, dst_nb2=1024, dst_nb3=0, q_type=mx.F32, dst_type=mx.F32, D=128, DV=128, T=2, H=8, KV=64, HK=2, S=1,
             scale=1.0, max_bias=0.0, softcap=0.0)
    a.update(kw)
    return mx.FaQArgs(**a)


U, A = "E_UNSUPPORTED", "E_ARG"
FA_REFUSALS = [(dict(D=48), U), (dict(D=0), U), (dict(DV=-32), U), (dict(D=576, DV=512), U), (dict(max_bias=8.0), U),
               (dict(k=dict(type=mx.F16)), U), (dict(v=dict(type=mx.Q4_K)), U), (dict(KV=1 << 30), U), (dict(T=1 << 20, H=4096), U),
               (dict(S=1 << 20, HK=8), U), (dict(KV=1 << 18, HK=1 << 9, H=1 << 9), U),
               (dict(q_dev=None), A), (dict(dst_dev=None), A), (dict(q_dev=FAKE + 8), A), (dict(dst_dev=FAKE + 8), A),
               (dict(k=dict(q_dev=None)), A), (dict(v=dict(d_dev=None)), A), (dict(k=dict(q_dev=FAKE + 8)), A),
               (dict(v=dict(d_dev=FAKE + 4)), A), (dict(k=dict(nb1=100)), A), (dict(v=dict(nb2=-128)), A), (dict(k=dict(nb3=16)), A),
               (dict(T=-1), A), (dict(S=-1), A), (dict(H=0), A), (dict(HK=0), A), (dict(HK=3), A), (dict(KV=-1), A),
               (dict(q_type=mx.BF16), A), (dict(dst_type=mx.Q8_0), A), (dict(q_nb1=130), A), (dict(q_type=mx.F16, q_nb1=132), A),
               (dict(dst_nb1=130), A), (dict(mask_nb1=60), A), (dict(mask_nb1=66), A), (dict(mask_nb3=2), A), (dict(mask_dev=FAKE + 4), A)]


@pytest.mark.parametrize("bad,why", FA_REFUSALS, ids=lambda b: b if isinstance(b, str) else "-".join(f"{k}={v}" for k, v in b.items()))
def test_attention_refusals(bad, why):
    L = mx.lib()
    a = fa(**bad)
    assert L.mi355x_flash_attn_q_workspace(ctypes.byref(a), 0) == 0
    assert L.mi355x_flash_attn_q(ctypes.byref(a), 0, FAKE, 1 << 40, None) == getattr(mx, why)


def test_attention_workspace_and_nothing_to_do():
    L = mx.lib()
    a = fa()
    need = L.mi355x_flash_attn_q_workspace(ctypes.byref(a), 0)
    assert need > 0
    assert L.mi355x_flash_attn_q(ctypes.byref(a), 0, FAKE, need - 1, None) == mx.E_NOMEM
    assert L.mi355x_flash_attn_q(ctypes.byref(a), 0, None, need, None) == mx.E_NOMEM
    assert L.mi355x_flash_attn_q(ctypes.byref(a), 0, FAKE + 16, need, None) == mx.E_NOMEM
    assert L.mi355x_flash_attn_q(ctypes.byref(a), 65, FAKE, 1 << 40, None) == mx.E_ARG
    assert L.mi355x_flash_attn_q(None, 0, FAKE, need, None) == mx.E_ARG
    for none in (dict(T=0), dict(S=0)):
        assert L.mi355x_flash_attn_q(ctypes.byref(fa(q_dev=None, dst_dev=None, **none)), 0, None, 0, None) == mx.OK


def test_binding_refusals():
    """Shapes, types and strides that the binding itself turns down."""
    q, d = torch.zeros(6, 2, 64, dtype=torch.int8), torch.zeros(6, 2, 2, dtype=torch.float16)
    c = mx.KvCache(mx.Q8_0, q, d)
    assert c.shape == (6, 2, 64) and c.permute(1, 0, 2).shape == (2, 6, 64) and c[1:4].shape == (3, 2, 64)
    for args in ((mx.Q8_0, q, None), (mx.Q4_0, q, d), (mx.Q8_0, q, d.float()), (mx.Q8_0, q, d[:, :, :1]), (mx.Q8_0, q[:, :, ::2], d[:, :, :1]),
                 (mx.Q8_0, q, d.transpose(0, 1).contiguous().transpose(0, 1)), (mx.F16, q.half(), d), (mx.Q4_K, q, d)):
        with pytest.raises(mx.MI355XError):
            mx.KvCache(*args)
    with pytest.raises(mx.MI355XError):
        mx.kv_cache(mx.Q4_0, 4, 48, device="cpu")
    x = torch.zeros(3, 2, 64)
    i = torch.zeros(3, dtype=torch.int64)
    for pairs, idx in (([(c, x[:, :1])], i), ([(c, x.double())], i), ([(c, x)], i.float()), ([(c, x)], i[:2]), ([(c, x)], i.view(1, 3)),
                       ([(c, x), (c, x[:2])], i)):
        with pytest.raises(mx.MI355XError):
            mx.set_rows(pairs, idx)
    kv = c.permute(1, 0, 2)
    qq, out = torch.zeros(4, 1, 64), torch.zeros(1, 4, 64)
    m = torch.zeros(1, 8, dtype=torch.float16)
    f16 = mx.KvCache(mx.F16, torch.zeros(2, 6, 64, dtype=torch.float16))
    for a in ((qq[None], kv, kv, m, out), (qq[..., :32], kv, kv, m, out), (qq.double(), kv, kv, m, out), (qq, kv[:, :5], kv, m, out),
              (qq, kv, kv, m.float(), out), (qq, kv, kv, m[:, :4], out), (qq, kv, kv, m, out[:, :, :32]), (qq, f16, kv, m, out),
              (qq, kv, f16, m, out), (torch.zeros(4, 1, 128)[..., ::2], kv, kv, m, out)):
        with pytest.raises(mx.MI355XError):
            mx.flash_attn_q_workspace(*a)

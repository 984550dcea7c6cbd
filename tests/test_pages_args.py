"""What the operators on a KV cache in pages refuse, before touching the device (CPU)."""
import ctypes

import pytest
import torch

import ggml_mi355x as mx

FAKE = 1 << 20      # aligned, never dereferenced on these paths
U, A, M = "E_UNSUPPORTED", "E_ARG", "E_NOMEM"


def step(**kw):
    a = dict(table_dev=FAKE, table_nb=8, n_past_dev=FAKE, n_new_dev=FAKE, parent_dev=None, parent_nb=0, n_table=8, S=2, T=3, page=64)
    a.update(kw)
    return mx.KvStepArgs(**a)


def rows(**kw):
    a = dict(type=mx.Q8_0, q_dev=FAKE, d_dev=FAKE, n_rows=1024, nb1=512, nb2=128, H=4, D=128, x_type=mx.F32, x_dev=FAKE, x_nb1=512, x_nb2=128)
    a.update(kw)
    return mx.KvRows(**a)


STEP_REFUSALS = [dict(S=-1), dict(T=-1), dict(page=0), dict(page=-32), dict(page=48), dict(n_table=-1), dict(n_table=0), dict(n_table=(1 << 23) + 1),
                 dict(table_nb=-1), dict(parent_nb=-1), dict(table_dev=None), dict(n_past_dev=None), dict(table_dev=FAKE + 2),
                 dict(n_past_dev=FAKE + 1), dict(n_new_dev=FAKE + 2), dict(parent_dev=FAKE + 2), dict(parent_dev=FAKE, T=65),
                 dict(S=1 << 12, T=(1 << 10) + 1), dict(page=2048)]
APPEND_REFUSALS = [dict(q_dev=None), dict(qr_dev=None), dict(q_dev=FAKE + 8), dict(qr_dev=FAKE + 4), dict(q_type=mx.Q8_0), dict(qr_type=mx.BF16),
                   dict(q_nb1=12), dict(q_nb3=-8), dict(qr_nb2=4), dict(H=0), dict(H=-4), dict(H=1 << 30), dict(k_nb3=4), dict(v_nb3=-8), dict(pos_nb=-1),
                   dict(pos_dev=FAKE + 2), dict(freq_dev=FAKE + 2), dict(freq_dev=None), dict(n_rot=12), dict(n_rot=-8), dict(n_rot=136),
                   dict(qr_dev=FAKE), dict(qr_dev=FAKE, neox=0, qr_type=mx.F16), dict(qr_dev=FAKE, neox=0, qr_nb1=1024)]
ROW_REFUSALS = [dict(type=mx.Q4_K), dict(q_dev=FAKE + 8), dict(d_dev=None), dict(nb1=500), dict(nb2=-128), dict(H=0), dict(D=48), dict(n_rows=63), dict(n_rows=-1),
                dict(H=1 << 14, D=256)]
ROW_X_REFUSALS = [dict(x_type=mx.BF16), dict(x_dev=None), dict(x_dev=FAKE + 4), dict(x_nb1=516), dict(x_nb2=-8)]


def names(b):
    return b if isinstance(b, str) else "-".join(f"{k}={v}" for k, v in b.items())


def append(step_kw=None, k=None, v=None, **kw):
    a = dict(step=step(**(step_kw or {})), k=rows(**(k or {})), v=rows(**{"q_dev": 2 * FAKE, **(v or {})}), k_nb3=2048, v_nb3=2048, q_dev=FAKE, q_nb1=512,
             q_nb2=128, q_nb3=2048, qr_dev=2 * FAKE, qr_nb1=512, qr_nb2=128, qr_nb3=2048, q_type=mx.F32, qr_type=mx.F32, H=4, freq_dev=FAKE, pos_dev=None,
             pos_nb=0, n_rot=128, neox=1, mscale=1.0)
    a.update(kw)
    return mx.KvAppendArgs(**a)


def call_append(a, err=None):
    return mx.lib().mi355x_kv_append(ctypes.byref(a), err, None)


@pytest.mark.parametrize("bad", STEP_REFUSALS, ids=names)
def test_steps(bad):
    assert call_append(append(bad)) == mx.E_ARG
    assert mx.lib().mi355x_kv_keep(ctypes.byref(step(**bad)), (mx.KvRows * 1)(rows()), 1, FAKE, 3, FAKE, 3, None, None) == mx.E_ARG
    a = attend(bad)
    assert mx.lib().mi355x_flash_attn_paged_workspace(ctypes.byref(a), 0) == 0
    assert mx.lib().mi355x_flash_attn_paged(ctypes.byref(a), 0, FAKE, 1 << 40, None, None) == mx.E_ARG


@pytest.mark.parametrize("bad", APPEND_REFUSALS, ids=names)
def test_append(bad):
    assert call_append(append(**bad)) == mx.E_ARG


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("bad", ROW_REFUSALS + ROW_X_REFUSALS, ids=names)
def test_append_rows(which, bad):
    assert call_append(append(**{which: bad})) == mx.E_ARG


def test_append_arguments_as_packed():
    """The binding packs mi355x_kv_append_args as the struct lies in memory."""
    a = append(pos_dev=FAKE, pos_nb=3, mscale=0.5)
    rest = (a.k_nb3, a.v_nb3, a.q_dev, a.q_nb1, a.q_nb2, a.q_nb3, a.qr_dev, a.qr_nb1, a.qr_nb2, a.qr_nb3, a.q_type, a.qr_type, a.H, a.freq_dev, a.pos_dev, a.pos_nb,
            a.n_rot, a.neox, a.mscale)
    row = lambda r: mx._KV_ROWS.pack(*[getattr(r, n) or 0 for n, _ in r._fields_])  # noqa: E731
    assert bytes(a.step) + row(a.k) + row(a.v) + mx._KV_APPEND.pack(*rest) == bytes(a)


def test_append_calls():
    assert mx.lib().mi355x_kv_append(None, None, None) == mx.E_ARG
    assert call_append(append(), FAKE + 2) == mx.E_ARG
    assert call_append(append(v=dict(q_dev=FAKE))) == mx.E_ARG                 # one cache twice
    assert call_append(append(v=dict(H=8))) == mx.E_ARG
    assert call_append(append(k=dict(D=96), n_rot=128)) == mx.E_ARG
    for none in (dict(S=0), dict(T=0)):
        assert call_append(append(none)) == mx.OK
        empty = dict(q_dev=None, d_dev=None, x_dev=None)
        assert call_append(append({**none, "table_dev": None, "n_past_dev": None, "n_table": 0}, empty, empty, q_dev=None, qr_dev=None, freq_dev=None)) == mx.OK


def test_keep():
    L = mx.lib()

    def keep(r=(rows(),), s=None, path=FAKE, nb=3, n=FAKE, A=3, err=None, n_out=None):
        return L.mi355x_kv_keep(ctypes.byref(s or step()), (mx.KvRows * len(r))(*r), len(r) if n_out is None else n_out, path, nb, n, A, err, None)

    for bad in ROW_REFUSALS:
        assert keep((rows(), rows(**{"q_dev": 2 * FAKE, **bad}))) == mx.E_ARG, bad
    assert keep(n_out=0) == mx.E_ARG and keep((rows(),) * 2) == mx.E_ARG
    assert keep(tuple(rows(q_dev=FAKE * (i + 1)) for i in range(5))) == mx.E_ARG
    assert keep(path=None) == mx.E_ARG and keep(path=FAKE + 2) == mx.E_ARG and keep(n=FAKE + 2) == mx.E_ARG and keep(err=FAKE + 2) == mx.E_ARG
    assert keep(nb=-1) == mx.E_ARG and keep(A=-1) == mx.E_ARG and keep(A=65) == mx.E_ARG
    assert L.mi355x_kv_keep(None, (mx.KvRows * 1)(rows()), 1, FAKE, 3, FAKE, 3, None, None) == mx.E_ARG
    assert L.mi355x_kv_keep(ctypes.byref(step()), None, 1, FAKE, 3, FAKE, 3, None, None) == mx.E_ARG
    assert keep(A=0, path=None) == mx.OK and keep(s=step(S=0)) == mx.OK and keep(s=step(T=0)) == mx.OK


def view(**kw):
    a = dict(type=mx.Q8_0, q_dev=FAKE, d_dev=FAKE, nb1=512, nb2=128, nb3=0)
    a.update(kw)
    return mx.KvView(**a)


def attend(step_kw=None, k=None, v=None, **kw):
    a = dict(step=step(**(step_kw or {})), q_dev=FAKE, q_nb1=1024, q_nb2=128, q_nb3=4096, k=view(**(k or {})), v=view(**(v or {})), n_rows=1024, dst_dev=FAKE,
             dst_nb1=128, dst_nb2=1024, dst_nb3=4096, q_type=mx.F32, dst_type=mx.F32, D=128, DV=128, H=8, HK=2, scale=1.0, softcap=0.0, max_kv=0)
    a.update(kw)
    return mx.FaPArgs(**a)


ATTEND_REFUSALS = [(dict(D=48), U), (dict(D=0), U), (dict(DV=-32), U), (dict(D=576, DV=512), U), (dict(D=256, DV=96), U), (dict(k=dict(type=mx.Q4_K)), U),
                   (dict(v=dict(type=mx.BF16)), U), (dict(k=dict(type=mx.F16)), U), (dict(v=dict(type=mx.F16)), U), (dict(step_kw=dict(S=1 << 20, T=1, n_table=1), HK=8), U), (dict(step_kw=dict(S=1, T=1 << 20), H=4096, HK=1), U),
                   (dict(q_dev=None), A), (dict(dst_dev=None), A), (dict(q_dev=FAKE + 8), A), (dict(dst_dev=FAKE + 8), A), (dict(k=dict(q_dev=None)), A),
                   (dict(v=dict(d_dev=None)), A), (dict(k=dict(q_dev=FAKE + 8)), A), (dict(v=dict(d_dev=FAKE + 4)), A), (dict(k=dict(nb1=100)), A),
                   (dict(v=dict(nb2=-128)), A), (dict(k=dict(nb1=1 << 24)), A), (dict(H=0), A), (dict(HK=0), A), (dict(HK=3), A), (dict(n_rows=-1), A),
                   (dict(n_rows=63), A), (dict(max_kv=-1), A), (dict(q_type=mx.BF16), A), (dict(dst_type=mx.Q8_0), A), (dict(q_nb1=130), A),
                   (dict(q_type=mx.F16, q_nb3=132), A), (dict(dst_nb1=130), A)]


@pytest.mark.parametrize("bad,why", ATTEND_REFUSALS, ids=names)
def test_attention(bad, why):
    L, a = mx.lib(), attend(**bad)
    assert L.mi355x_flash_attn_paged_workspace(ctypes.byref(a), 0) == 0
    assert L.mi355x_flash_attn_paged(ctypes.byref(a), 0, FAKE, 1 << 40, None, None) == getattr(mx, why)


def test_attention_workspace_and_nothing_to_do():
    L, a = mx.lib(), attend()
    need = L.mi355x_flash_attn_paged_workspace(ctypes.byref(a), 0)
    assert need > 0
    for ws, n, nsplit, err, why in ((FAKE, need - 1, 0, None, M), (None, need, 0, None, M), (FAKE + 16, need, 0, None, M), (FAKE, 1 << 40, 65, None, A),
                                    (FAKE, need, 0, FAKE + 2, A)):
        assert L.mi355x_flash_attn_paged(ctypes.byref(a), nsplit, ws, n, err, None) == getattr(mx, why)
    assert L.mi355x_flash_attn_paged(None, 0, FAKE, need, None, None) == mx.E_ARG
    for none in (dict(T=0), dict(S=0)):
        b = attend(none, q_dev=None, dst_dev=None)
        assert L.mi355x_flash_attn_paged_workspace(ctypes.byref(b), 0) > 0
        assert L.mi355x_flash_attn_paged(ctypes.byref(b), 0, None, 0, None, None) == mx.OK
    # the plan follows max_kv, not the table
    short = L.mi355x_flash_attn_paged_workspace(ctypes.byref(attend(dict(n_table=1 << 12), max_kv=300)), 0)
    assert short < L.mi355x_flash_attn_paged_workspace(ctypes.byref(attend(dict(n_table=1 << 12))), 0)


def test_binding_refusals():
    """Shapes, types and strides that the binding itself turns down."""
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    good = dict(table=i(2, 4), n_past=i(2), T=3, page=32)
    for bad in (dict(table=torch.zeros(2, 4)), dict(table=i(2, 8)[:, ::2]), dict(n_past=i(3)), dict(n_past=i(2, 1)), dict(n_past=i(4)[::2]), dict(page=16), dict(page=0),
                dict(T=-1), dict(n_new=i(1)), dict(n_new=i(2).long()), dict(parents=i(2, 4)), dict(parents=i(3, 3)), dict(parents=i(2, 65), T=65)):
        with pytest.raises(mx.MI355XError):
            mx.KvStep(**{**good, **bad})
    st = mx.KvStep(**good)
    with pytest.raises(mx.MI355XError):
        st.n_past = i(2)             # the address of the first would stay in use
    for bad in (dict(freq=torch.zeros(6)), dict(freq=torch.zeros(8).double()), dict(freq=torch.zeros(16)[::2]), dict(freq=torch.zeros(8), positions=torch.zeros(2, 3)),
                dict(freq=torch.zeros(8), positions=i(6))):
        with pytest.raises(mx.MI355XError):
            mx.Rope(**bad)
    assert torch.equal(mx.rope_freqs(4, 100.0, factors=[1.0, 2.0], device="cpu"), torch.tensor([1.0, 0.05]))
    kc, vc = mx.kv_cache(mx.Q8_0, 128, 2, 64, device="cpu"), mx.kv_cache(mx.Q4_0, 128, 2, 32, device="cpu")
    k, v, q = torch.zeros(2, 3, 2, 64), torch.zeros(2, 3, 2, 32), torch.zeros(2, 3, 4, 64)
    rope = mx.Rope(torch.zeros(32))
    for a, kw in (((kc, vc, k[:, :2], v), {}), ((kc, vc, k, v[..., :16]), {}), ((kc, vc, k.double(), v), {}), ((kc, vc, k, v), dict(q=q[:1])),
                  ((kc, vc, k, v), dict(q=q[..., :32])), ((kc, vc, k, v), dict(q=q, q_out=q[:, :, :2])), ((kc, vc, k, v), dict(q=q.double())), ((kc, vc, k, v), dict(q_out=q)),
                  ((kc[:, 0], vc, k, v), {}), ((kc, vc, k, v), dict(rope=mx.Rope(torch.zeros(32), positions=i(2, 4)))), ((kc, vc, k, v), dict(rope=rope))):
        with pytest.raises(mx.MI355XError):
            mx.kv_append(st, *a, **kw)
    for caches, path, kw in (([], i(2, 2), {}), ([kc] * 5, i(2, 2), {}), ([kc], i(3, 2), {}), ([kc], i(2, 2).long(), {}), ([kc], i(4), {}), ([kc], i(2, 4)[:, ::2], {}),
                             ([kc], i(2, 2), dict(n_keep=i(3))), ([kc], i(2, 2), dict(n_keep=torch.zeros(2)))):
        with pytest.raises(mx.MI355XError):
            mx.kv_keep(st, caches, path, **kw)
    qv, out = q.permute(0, 2, 1, 3), torch.zeros(2, 3, 4, 32)
    for a in ((qv[:1], kc, vc, st, out), (qv[:, :, :2], kc, vc, st, out), (qv[..., :32], kc, vc, st, out), (qv, kc[:64], vc, st, out), (qv, kc, kc, st, out),
              (qv, kc, vc, st, out.double()), (qv, kc, vc, st, torch.zeros(2, 4, 3, 32)), (qv.double(), kc, vc, st, out), (q[0], kc, vc, st, out)):
        with pytest.raises(mx.MI355XError):
            mx.flash_attn_paged_workspace(*a)

"""The quantized cache's calls with nothing to do: attention of no query rows or no sequences (CPU; the refusals' own
operands, never dereferenced), rows of no cache."""
import ctypes

import pytest

import ggml_mi355x as mx
from test_kv_args import FAKE, fa


@pytest.mark.parametrize("form", ["1", "0", ""], ids=["direct", "decoded", "chosen"])
@pytest.mark.parametrize("nsplit", [0, 1, 64])
@pytest.mark.parametrize("none", [dict(T=0), dict(S=0), dict(T=0, S=0), dict(T=0, KV=0), dict(S=0, KV=8), dict(T=0, KV=1 << 18, mask_nb1=1 << 18)],
                         ids=lambda d: "-".join(f"{k}{v}" for k, v in d.items()))
def test_workspace_of_nothing(monkeypatch, form, nsplit, none):
    """A workspace may be asked for before the shapes are looked at: some small size, and no error."""
    monkeypatch.setenv("MI355X_FA_Q_DIRECT", form)
    L = mx.lib()
    a = fa(**none)
    need = L.mi355x_flash_attn_q_workspace(ctypes.byref(a), nsplit)
    assert 0 < need <= 4096
    for ws, n in ((None, 0), (FAKE, need)):
        assert L.mi355x_flash_attn_q(ctypes.byref(a), nsplit, ws, n, None) == mx.OK


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["1", "0", ""], ids=["direct", "decoded", "chosen"])
@pytest.mark.parametrize("lead,T", [((), 0), ((3,), 0), ((0,), 2)])
def test_attention_of_nothing(torch_cuda, monkeypatch, form, lead, T):
    """The binding's own workspace too; no output value exists to be written."""
    import torch
    monkeypatch.setenv("MI355X_FA_Q_DIRECT", form)
    H, HK, KV, D = 4, 2, 40, 64
    kc, vc = mx.kv_cache(mx.Q8_0, *lead, HK, KV, D), mx.kv_cache(mx.Q4_0, *lead, HK, KV, D)
    q = torch.zeros(*lead, H, T, D, device="cuda")
    out = mx.flash_attn_q(q, kc, vc, None, 0.125)
    assert out.shape == (*lead, T, H, D)
    torch.cuda.synchronize()


def test_no_caches():
    for f in (lambda: mx.set_rows([]), lambda: mx.get_rows([])):
        with pytest.raises(mx.MI355XError):
            f()
    import torch
    c = mx.kv_cache(mx.Q8_0, 4, 2, 64, device="cpu")
    x = torch.zeros(2, 2, 64)
    with pytest.raises(mx.MI355XError):
        mx.set_rows([(c, x)] * 5)

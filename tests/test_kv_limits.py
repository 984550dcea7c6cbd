"""The largest attention calls over a quantized cache: what passes the count of a launch's threads is turned down before
anything is launched (CPU: no GPU, so a call that is taken fails where it launches)."""
import ctypes

import pytest

import ggml_mi355x as mx
from test_kv_args import FAKE, fa


def status(nsplit, **kw):
    a = fa(T=1, H=1, HK=1, mask_dev=None, **kw)
    need = mx.lib().mi355x_flash_attn_q_workspace(ctypes.byref(a), nsplit)
    return need, mx.lib().mi355x_flash_attn_q(ctypes.byref(a), nsplit, None, 0, None)


@pytest.mark.parametrize("DV,S,nsplit,taken", [(256, 1 << 20, 2, False), (256, (1 << 20) - 1, 2, True), (224, 1 << 20, 2, False), (128, 1 << 20, 2, True),
                                               (256, 1 << 21, 1, True), (256, 1 << 21, 0, True), (256, (1 << 21) + 1, 1, False),
                                               (64, 1 << 15, 64, True), (64, (1 << 15) + 1, 64, False)])
def test_row_tiles_and_splits(monkeypatch, DV, S, nsplit, taken):
    """The second launch has 256 threads for every row tile and 16 dims, fewer than 2^32 in all."""
    monkeypatch.setenv("MI355X_FA_Q_DIRECT", "1")
    need, st = status(nsplit, D=256 if DV > 128 else DV, DV=DV, S=S, KV=4096, k=dict(nb1=256, nb2=256), v=dict(nb1=256, nb2=256))
    assert (need > 0) == taken and st == (mx.E_NOMEM if taken else mx.E_UNSUPPORTED)

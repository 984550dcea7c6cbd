"""from_pages: a caller's choice, call by call, that a chain over a quantized cache in pages is not decoded first."""
import ctypes

import numpy as np
import pytest

import ggml_mi355x as lib
from test_pages_args import attend
from test_pages_gpu import MIXES, Q4_0, Q8_0, attend_case, cpu, gpu, ids, mx  # noqa: F401
from test_pages_norm import check


def test_workspace(monkeypatch):
    """It needs none of the decoded cache, and no environment variable changes that."""
    a = [attend(dict(S=1, T=512, n_table=128), max_kv=8192, from_pages=i) for i in (0, 1)]
    need = lambda x: lib.lib().mi355x_flash_attn_paged_workspace(ctypes.byref(x), 0)  # noqa: E731
    assert need(a[0]) > 2 * 2 * 8192 * 128 * 2 > need(a[1]) > 0
    monkeypatch.setenv("MI355X_FA_Q_DIRECT", "0")
    assert need(a[0]) > 2 * 2 * 8192 * 128 * 2 > need(a[1]) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("mix", MIXES, ids=ids)
def test_from_pages(mx, monkeypatch, mix):  # noqa: F811
    """The bits of the direct form, and its bound, where the library decodes first."""
    import torch
    c = attend_case(mx, *mix, (1, 300, False, [3900], 64, 8, 2, 128, 128))
    c["q"] = 3 * c["q"]
    q, caches, scale = gpu(c["q"]).permute(0, 2, 1, 3), [x[0] for x in c["caches"]], float(np.float32(128 ** -0.5))
    out = torch.zeros(1, 300, 8, 128, device="cuda")
    ws = torch.empty(mx.flash_attn_paged_workspace(q, *caches, c["step"], out, from_pages=True), dtype=torch.uint8, device="cuda")
    monkeypatch.setenv("MI355X_FA_Q_DIRECT", "1")
    direct = cpu(mx.flash_attn_paged(q, *caches, c["step"], scale))
    monkeypatch.setenv("MI355X_FA_Q_DIRECT", "0")
    decoded = cpu(mx.flash_attn_paged(q, *caches, c["step"], scale))
    got = cpu(mx.flash_attn_paged(q, *caches, c["step"], scale, out=out, workspace=ws, from_pages=True))
    assert np.array_equal(got, direct) and not np.array_equal(got, decoded)
    check(c, got, scale)

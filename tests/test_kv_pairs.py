"""SET_ROWS and GET_ROWS turn down calls whose outputs would overwrite each other (CPU)."""
import pytest
import torch

import ggml_mi355x as mx
from test_kv_args import FAKE, rows


def call(fn, *r, n=3):
    return getattr(mx.lib(), fn)((mx.KvRows * len(r))(*r), len(r), FAKE, mx.I64, n, None, None)


@pytest.mark.parametrize("others", [0, 1, 2])
def test_one_destination_twice(others):
    """The order in which two outputs of a call are written is not defined: no two of them start at one address."""
    far = [rows(q_dev=FAKE * (5 + i), x_dev=FAKE * (9 + i)) for i in range(others)]
    a, b = rows(q_dev=FAKE, x_dev=FAKE * 2), rows(q_dev=FAKE, x_dev=FAKE * 3, type=mx.Q4_0)
    assert call("mi355x_set_rows", a, *far, b) == mx.E_ARG
    a, b = rows(q_dev=FAKE, x_dev=FAKE * 2), rows(q_dev=FAKE * 4, x_dev=FAKE * 2, x_type=mx.F16)
    assert call("mi355x_get_rows", a, *far, b) == mx.E_ARG
    # sources may be shared, and with no rows there is nothing to overwrite
    assert call("mi355x_set_rows", rows(q_dev=None, d_dev=None, x_dev=None), rows(q_dev=None, d_dev=None, x_dev=None), n=0) == mx.OK


@pytest.mark.gpu
def test_one_source_twice(torch_cuda):
    """One tensor into two caches, and one cache read twice."""
    x = torch.randn(3, 2, 64, device="cuda")
    a, b = mx.kv_cache(mx.Q8_0, 5, 2, 64), mx.kv_cache(mx.Q4_0, 5, 2, 64)
    mx.set_rows([(a, x), (b, x)])
    y, h = mx.get_rows([a, a], out=[torch.empty(5, 2, 64, device="cuda"), torch.empty(5, 2, 64, device="cuda", dtype=torch.float16)])
    assert torch.equal(y.half(), h) and float((y[:3] - x).abs().max()) <= float(x.abs().max()) / 127
    assert float((mx.get_rows([b])[0][:3] - x).abs().max()) <= float(x.abs().max()) / 8 * 1.01

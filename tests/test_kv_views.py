"""KvCache indexing gives views and nothing else: what a store writes through one is in the cache (CPU)."""
import numpy as np
import pytest
import torch

import ggml_mi355x as mx


def cache(t=mx.Q4_0):
    return mx.kv_cache(t, 6, 2, 64, device="cpu")


@pytest.mark.parametrize("t", [mx.Q8_0, mx.Q4_0, mx.F16])
@pytest.mark.parametrize("at", [slice(2, 5), slice(None), slice(0, 6, 2), 3, -1, (slice(1, 3), 1), (2, slice(0, 1)), np.int64(4)],
                         ids=lambda a: str(a).replace(" ", ""))
def test_views(t, at):
    c = cache(t)
    v = c[at]
    assert v.q.untyped_storage().data_ptr() == c.q.untyped_storage().data_ptr()
    assert v.shape == torch.zeros(6, 2, 64)[at].shape
    if t != mx.F16:
        assert v.d.untyped_storage().data_ptr() == c.d.untyped_storage().data_ptr()


@pytest.mark.parametrize("at", [torch.tensor([0, 2]), [0, 2], torch.tensor([True] * 6), True, np.array([1, 2]), torch.tensor(1), None,
                                Ellipsis, (slice(None), [0]), (slice(None), torch.tensor([1])), (slice(None), True), (0, None),
                                (0, 0, slice(None)), (slice(None), slice(None), slice(0, 32)), 1.0, "0"], ids=lambda a: str(a).replace(" ", "")[:30])
def test_what_would_be_a_copy_or_no_view_of_leading_dims(at):
    with pytest.raises(mx.MI355XError):
        cache()[at]

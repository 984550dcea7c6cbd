"""Chains over a cache in pages with a key or value that is no number: it reaches exactly the tokens that see it, in every form."""
import numpy as np
import pytest

import pages_oracle as P
from test_pages_gpu import ATTENDED, F16, NAME, cache_of, cpu, form, gpu, i32, mx, tables, zeros_i32  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [0x7E00, 0x7C00, 0xFC00], ids=["nan", "inf", "minus_inf"])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("D,DV", [(64, 64), (128, 64), (192, 128), (96, 128), (256, 256)])
@pytest.mark.parametrize("kt,vt", ATTENDED, ids=lambda t: NAME[t])
def test_exactly_the_rows_that_see_it(mx, form, kt, vt, D, DV, which, bits):  # noqa: F811
    """In the last block of a head's dims of one new token (the 20th of 37, of the 3rd head), of one held row and of one that no sequence has."""
    T, page, H, HK, past = 37, 32, 6, 3, [75, 40, 3]
    rng = np.random.default_rng(D + DV)
    new = [T, T, 30]
    table, pages = tables(rng, past, new, page)
    caches = [cache_of(mx, t, pages * page, HK, d, rng) for t, d in ((kt, D), (vt, DV))]
    i = "kv".index(which)
    at = [P.row(table[0], page, past[0] + 19), P.row(table[1], page, 21), P.row(table[2], page, past[2] + 30)]
    plane = caches[i][1][-1].copy()
    plane[at, 2, -1] = bits                          # the last scale, or the last value of an F16 cache
    c = caches[i][0]
    (c.q if c.type == F16 else c.d).copy_(gpu(plane.view(np.float16)))
    q = rng.standard_normal((3, T, H, D)).astype(np.float32)
    err = zeros_i32()
    step = mx.KvStep(i32(table), i32(past), T, page, n_new=i32(new))
    got = cpu(mx.flash_attn_paged(gpu(q).permute(0, 2, 1, 3), caches[0][0], caches[1][0], step, D ** -0.5, err=err))
    sees = np.zeros(got.shape[:3], bool)
    sees[0, 19:, 4:] = sees[1, :, 4:] = True         # heads 4 and 5 are the third key head's
    if which == "v" and vt == F16:                   # that dim at least: P times an infinity is one
        assert not np.isfinite(got[sees][:, -1]).any()
    elif which == "k" and kt == F16 and bits != 0x7E00:
        assert not np.isfinite(got[0, 19:, 4:]).all()    # scores of either sign, infinite
    else:                                            # a scale stands for its key's whole row
        assert np.isnan(got[sees]).all()
    for s in range(3):                               # all others are what they are without it
        want, tol = P.attend(q[s].transpose(1, 0, 2).astype(np.float64), caches[0][1], caches[1][1], kt, vt, table[s], page, pages, past[s], new[s], None, D ** -0.5)
        d = np.abs(got[s] - want)[~sees[s]]
        assert np.isfinite(d).all() and (d <= tol[~sees[s]] + 1e-30).all()
    assert int(err) == 0

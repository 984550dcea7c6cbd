"""Attention over a cache in pages held to its roundings (pages_norm; kv_norm where the cache is decoded first): a missing key tile, one counted twice or an
operand rounded once more is noticed, at thousands of keys, many pages and every split."""
import numpy as np
import pytest

import kv_norm
import kv_oracle as R
import pages_norm as N
import pages_oracle as P
from test_pages_gpu import ATTENDED, F16, NAME, Q4_0, Q8_0, attend_case, cache_of, cpu, gpu, i32, ids, mx, tables  # noqa: F401

pytestmark = pytest.mark.gpu


def held(c, s):
    """K, V [HK][n][dims] of sequence s and their blocks' scales (None: F16)."""
    n = c["past"][s] + c["new"][s]
    at = [P.row(c["table"][s], c["page"], j) for j in range(n)]
    values, scales = [], []
    for (_, pl), t in zip(c["caches"], (c["kt"], c["vt"])):
        pl = [p[at] for p in pl]
        values.append(P.cache_values(pl, t).transpose(1, 0, 2))
        scales.append(None if t == F16 else pl[1].view(np.float16).astype(np.float64).transpose(1, 0, 2))
    return values, scales


def check(c, got, scale, softcap=0.0, half=False, decoded=False):
    errors, total, limit = [], 0.0, 0.0
    for s in range(c["S"]):
        n = c["new"][s]
        assert not got[s, n:].any()
        if not n:
            continue
        (k, v), (kd, vd) = held(c, s)
        q = c["q"][s, :n].transpose(1, 0, 2).astype(np.float64)
        mask = N.mask_of(c["past"][s], n, n, None if c["parents"] is None else c["parents"][s])
        if decoded:
            want, lim = kv_norm.attention(q, k, v, mask, scale, softcap, vd=vd, half_out=half)
            sigma = lim / kv_norm.SIGMAS
        else:
            want, sigma = N.attention(q, k, v, mask, scale, softcap, kd, vd, c["kt"], c["q"].dtype == np.float16, half)
        d = got[s, :n].astype(np.float64) - want
        errors.append(N.errors(got[s, :n], want, sigma)[0])
        total, limit = total + (d ** 2).sum(), limit + (sigma ** 2).sum()
    assert max(errors) <= 1 and total <= 1.1 ** 2 * limit, (errors, float(np.sqrt(total / limit)))


LONG = [  # S, T, tree, past, page, H, HK, D, DV, softcap, half
    (1, 1, False, [5000], 128, 32, 8, 128, 128, 0.0, False),
    (2, 5, True, [4100, 2399], 32, 8, 2, 128, 128, 5.0, True),
    (3, 16, True, [3000, 33, 0], 96, 8, 2, 64, 64, 0.0, False),
    (1, 16, True, [2600], 32, 4, 2, 256, 256, 0.0, True),
    (2, 40, False, [0, 2000], 256, 4, 1, 160, 128, 0.0, False),
    (1, 70, False, [2500], 64, 8, 2, 192, 128, 30.0, True),
    (4, 33, False, [0, 31, 800, 3333], 32, 8, 2, 64, 64, 0.0, True),
]


@pytest.mark.parametrize("nsplit", [0, 1, 2, 7, 64])
@pytest.mark.parametrize("kt,vt", ATTENDED, ids=lambda t: NAME[t])
@pytest.mark.parametrize("case", LONG, ids=lambda c: "S%dT%d%sD%d-%d" % (c[0], c[1], "t" if c[2] else "c", c[7], c[8]))
def test_every_key_counts_once(mx, monkeypatch, kt, vt, case, nsplit):  # noqa: F811
    import torch
    *shape, softcap, half = case
    c = attend_case(mx, kt, vt, tuple(shape), seed=nsplit)
    c["q"] = (3 * c["q"]).astype(np.float16 if half else np.float32)     # scores some 3 apart, so that a rounded Q weighs more than P
    scale = float(np.float32(c["D"] ** -0.5))
    q = gpu(c["q"]).permute(0, 2, 1, 3)
    for direct, rows in (("1", "16"), ("1", "32"), ("0", "")):
        if direct == "0" and (kt == F16 or c["parents"] is not None):
            continue
        monkeypatch.setenv("MI355X_FA_Q_DIRECT", direct)
        monkeypatch.setenv("MI355X_FA_Q_ROWS", rows)
        out = torch.full((c["S"], c["T"], c["H"], c["DV"]), float("nan"), device="cuda", dtype=torch.float16 if half else torch.float32)
        mx.flash_attn_paged(q, *[x[0] for x in c["caches"]], c["step"], scale, softcap=softcap, nsplit=nsplit, out=out)
        check(c, cpu(out), scale, softcap, half, decoded=direct == "0")

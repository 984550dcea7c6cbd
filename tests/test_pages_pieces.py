"""Long chains over long quantized caches in pages, decoded first: the workspace does not grow with tokens times keys, and tokens that go through in several
pieces are as those of one."""
import ctypes

import numpy as np
import pytest

import ggml_mi355x as lib
import kv_norm
import pages_oracle as P
from test_pages_args import attend
from test_pages_gpu import Q4_0, Q8_0, cache_of, cpu, gpu, i32, mx, tables, zeros_i32  # noqa: F401


@pytest.mark.parametrize("T,max_kv", [(512, 131072), (4096, 131072), (65536, 131072), (1 << 20, 65536), (1 << 20, 2048)])
def test_workspace(monkeypatch, T, max_kv):
    """Decoded K and V, 128 MiB, and what the tokens themselves take: partial rows of at most 16 splits and a byte for 32 tokens and 64 keys."""
    monkeypatch.setenv("MI355X_FA_Q_DIRECT", "0")
    H, HK, D = 8, 2, 128
    a = attend(dict(S=1, T=T, n_table=1 << 12), max_kv=max_kv)
    need = lib.lib().mi355x_flash_attn_paged_workspace(ctypes.byref(a), 0)
    assert 2 * HK * max_kv * D * 2 < need <= 2 * HK * max_kv * D * 2 + (1 << 27) + 16 * T * H * (D + 2) * 4 + T // 32 * (max_kv // 64 + 16) + 4096


@pytest.mark.gpu
@pytest.mark.parametrize("kt,vt,H,HK,D,DV,half", [(Q8_0, Q4_0, 2, 1, 64, 64, False), (Q4_0, Q8_0, 4, 2, 128, 96, True)])
def test_pieces(mx, monkeypatch, kt, vt, H, HK, D, DV, half):  # noqa: F811
    """4100 tokens, 4090 of them real, on 12310 keys with room for 16800: two pieces; a sequence without tokens and a short one beside it."""
    import torch
    monkeypatch.setenv("MI355X_FA_Q_DIRECT", "0")
    T, page, max_kv = 4100, 96, 16800
    rng = np.random.default_rng(D)
    past, new = [12310, 50, 7], [4090, 0, 4081]
    table, pages = tables(rng, past, new, page)
    caches = [cache_of(mx, t, pages * page, HK, d, rng) for t, d in ((kt, D), (vt, DV))]
    q = torch.randn(3, T, H, D, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(torch.float16 if half else torch.float32)
    table = np.concatenate([table, np.full((3, max_kv // page + 1 - table.shape[1]), -1, np.int32)], 1)
    step = mx.KvStep(i32(table), i32(past), T, page, n_new=i32(new))
    err = zeros_i32()
    out = torch.full((3, T, H, DV), float("nan"), device="cuda", dtype=torch.float16 if half else torch.float32)
    mx.flash_attn_paged(q.permute(0, 2, 1, 3), caches[0][0], caches[1][0], step, D ** -0.5, out=out, max_kv=max_kv, err=err)
    got = cpu(out)
    assert int(err) == 0
    cut = (1 << 26) // ((max_kv + 63) // 64 * 64) // 32 * 32
    assert 64 < cut < T - 64
    rows = sorted({0, 1, 31, 32, 33, 2000, *range(cut - 34, cut + 34), *range(4040, 4100)})
    for s in range(3):
        n = past[s] + new[s]
        real = [t for t in rows if t < new[s]]
        assert not got[s, new[s]:].any()
        if not real:
            continue
        at = [P.row(table[s], page, j) for j in range(n)]
        k, v = (P.cache_values([p[at] for p in pl], t).transpose(1, 0, 2) for (_, pl), t in zip(caches, (kt, vt)))
        mask = np.where(np.arange(n) <= past[s] + np.array(real)[:, None], 0.0, -np.inf)
        vd = caches[1][1][1][at].view(np.float16).transpose(1, 0, 2)
        want, limit = kv_norm.attention(cpu(q)[s, real].transpose(1, 0, 2), k, v, mask, D ** -0.5, vd=vd, half_out=half)
        assert kv_norm.ratio(got[s, real], want, limit) <= 1

"""Chains over a quantized cache in pages, decoded first, captured once: every replay follows the lengths, tables and tokens that lie on the device then, with
eager calls on the same workspace in between."""
import numpy as np
import pytest

import kv_norm
import pages_oracle as P
from test_pages_gpu import Q4_0, Q8_0, cache_of, cpu, gpu, i32, mx, zeros_i32  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kt,vt,nsplit", [(Q8_0, Q8_0, 0), (Q4_0, Q8_0, 3)])
def test_replays(mx, monkeypatch, kt, vt, nsplit):  # noqa: F811
    import torch
    monkeypatch.setenv("MI355X_FA_Q_DIRECT", "0")
    S, T, H, HK, D, page, n_table = 2, 70, 4, 2, 128, 32, 60
    rng = np.random.default_rng(3)
    pages = S * n_table
    (kc, kp), (vc, vp) = cache_of(mx, kt, pages * page, HK, D, rng), cache_of(mx, vt, pages * page, HK, D, rng)
    table, past, new = i32(np.zeros((S, n_table))), i32([0, 0]), i32([1, 1])
    q, out, err = torch.zeros(S, T, H, D, device="cuda"), torch.zeros(S, T, H, D, device="cuda"), zeros_i32()
    step = mx.KvStep(table, past, T, page, n_new=new)
    qv = q.permute(0, 2, 1, 3)
    ws = torch.empty(mx.flash_attn_paged_workspace(qv, kc, vc, step, out, nsplit), dtype=torch.uint8, device="cuda")

    def call():
        mx.flash_attn_paged(qv, kc, vc, step, D ** -0.5, nsplit=nsplit, out=out, workspace=ws, err=err)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call()
    for i in range(8):
        tab = rng.permutation(pages).reshape(S, n_table).astype(np.int32)
        p = [int(x) for x in (rng.integers(0, n_table * page - T, S) if i % 3 else rng.integers(0, 70, S))]
        n = [[T, 0], [1, T], [33, 64], [T, T]][i % 4]
        x = rng.standard_normal((S, T, H, D)).astype(np.float32)
        for d, y in ((table, tab), (past, np.array(p, np.int32)), (new, np.array(n, np.int32)), (q, x)):
            d.copy_(gpu(y))
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        if i in (2, 5):
            call()
        else:
            graph.replay()
        got = cpu(out)
        assert int(err) == 0
        for s in range(S):
            assert not got[s, n[s]:].any()
            if not n[s]:
                continue
            at = [P.row(tab[s], page, j) for j in range(p[s] + n[s])]
            k, v = (P.cache_values([y[at] for y in pl], t).transpose(1, 0, 2) for pl, t in ((kp, kt), (vp, vt)))
            mask = np.where(np.arange(len(at)) <= p[s] + np.arange(n[s])[:, None], 0.0, -np.inf)
            want, limit = kv_norm.attention(x[s, :n[s]].transpose(1, 0, 2), k, v, mask, D ** -0.5, vd=vp[1][at].view(np.float16).transpose(1, 0, 2))
            assert kv_norm.ratio(got[s, :n[s]], want, limit) <= 1

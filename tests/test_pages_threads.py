"""First calls of every kernel over pages from several host threads at once, a stream and a workspace each."""
import threading

import numpy as np
import pytest

from test_pages_gpu import F16, Q4_0, Q8_0, attend_case, cpu, gpu, mx  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("direct", ["1", "0"], ids=["direct", "decoded"])
def test_first_calls_of_threads(mx, monkeypatch, direct):  # noqa: F811
    import torch
    monkeypatch.setenv("MI355X_FA_Q_DIRECT", direct)
    work = []
    for t in ((Q8_0, Q8_0), (Q4_0, Q4_0), (F16, F16)):
        for D, DV in ((64, 64), (128, 128), (192, 128), (256, 256)):
            c = attend_case(mx, *t, (2, 20, False, [100, 300], 32, 4, 2, D, DV), seed=D)
            work.append((gpu(c["q"]).permute(0, 2, 1, 3), [x[0] for x in c["caches"]], c["step"], D ** -0.5))
    results, failed = [None] * 4, []
    gate = threading.Barrier(4)
    torch.cuda.synchronize()

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                gate.wait()
                outs = [mx.flash_attn_paged(q, *kv, step, scale) for q, kv, step, scale in work]
                torch.cuda.current_stream().synchronize()
            results[i] = [cpu(o) for o in outs]
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not failed
    again = [cpu(mx.flash_attn_paged(q, *kv, step, scale)) for q, kv, step, scale in work]
    assert all(np.array_equal(x, y) for r in results for x, y in zip(r, again))

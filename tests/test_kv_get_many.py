"""GET_ROWS of more blocks than one launch takes, and of one block: every row by its own index."""
import pytest

from test_kv_gpu import TYPES, ids, mx, noisy_cache  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", TYPES, ids=ids)
@pytest.mark.parametrize("n,H,D,wide", [((1 << 18) + 333, 8, 256, False), ((1 << 19) - 1, 8, 128, True), (1, 1, 32, False), (1 << 18, 8, 256, True)])
def test_rows_in_several_launches(mx, t, n, H, D, wide):
    """Two caches of different widths as fp16 and F32, indices repeated, some outside (their rows stay as they were)."""
    import torch
    rows = 100
    a, b = noisy_cache(mx, t, rows, H, D), noisy_cache(mx, t, rows, H * 32, seed=2)
    g = torch.Generator(device="cuda").manual_seed(n)
    at = torch.randint(0, rows, (n,), generator=g, device="cuda", dtype=torch.int64 if wide else torch.int32)
    at[-1] = rows - 1
    whole = mx.get_rows([a, b])
    x, y = torch.full((n, H, D), 7.0, device="cuda", dtype=torch.float16), torch.full((n, H * 32), 7.0, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    bad = torch.arange(min(3, n), n, 70001, device="cuda")
    at[bad] = rows
    mx.get_rows([a, b], at, out=[x, y], err=err)
    assert int(err) == int(n > 3)
    at[bad] = 0
    step = 1 << 16
    for i in range(0, n, step):
        j = at[i:i + step].long()
        here = bad[(bad >= i) & (bad < i + step)] - i
        for got, want in ((x, whole[0].half()), (y, whole[1])):
            w = want[j]
            w[here] = 7.0
            assert torch.equal(got[i:i + step], w), i

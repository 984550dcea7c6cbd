"""SET_ROWS, GET_ROWS and FLASH_ATTN_EXT of a quantized KV cache on the GPU, against plain numpy:
stored bits equal to the formats' definition, read values exact, attention within the bound that
fp16 operands allow (kv_oracle.attention)."""
import numpy as np
import pytest

import kv_oracle as R

pytestmark = pytest.mark.gpu

Q4_0, Q8_0 = R.Q4_0, R.Q8_0
TYPES = [Q8_0, Q4_0]
MIXES = [(Q8_0, Q8_0), (Q4_0, Q4_0), (Q8_0, Q4_0), (Q4_0, Q8_0)]
NAME = {Q8_0: "q8_0", Q4_0: "q4_0"}
INF = float("inf")


def ids(v):
    return NAME.get(v) if not isinstance(v, tuple) else "-".join(NAME[t] for t in v)


@pytest.fixture(scope="module")
def mx(torch_cuda):
    import ggml_mi355x
    ggml_mi355x.lib()
    return ggml_mi355x


@pytest.fixture(params=["1 16", "1 32", "0 ", " "], ids=["direct", "direct32", "decoded", "chosen"])
def form(request, monkeypatch):
    """Attention tests run under every form (the kernel that reads the cache as it is stored, with 16 and, at head
    dims up to 64, with 32 rows a wave; the cache decoded to fp16 first, which is the fp16 kernel's arithmetic) and the library's
    choice per call."""
    direct, rows = request.param.split(" ")
    monkeypatch.setenv("MI355X_FA_Q_DIRECT", direct)
    monkeypatch.setenv("MI355X_FA_Q_ROWS", rows)


def gpu(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def cpu(t):
    import torch
    torch.cuda.synchronize()
    return t.cpu().numpy()


def noisy_cache(mx, t, *shape, seed=1):
    """A cache whose every byte is random (finite scales)."""
    import torch
    c = mx.kv_cache(t, *shape)
    g = torch.Generator(device="cuda").manual_seed(seed)
    c.q.view(torch.uint8).random_(0, 256, generator=g)
    c.d.uniform_(0.001, 0.1, generator=g)
    return c


# ---- SET_ROWS -------------------------------------------------------------------------------

@pytest.mark.parametrize("t", TYPES, ids=ids)
@pytest.mark.parametrize("n,H,D", [(1, 8, 128), (2, 1, 32), (37, 3, 96), (300, 8, 64), (1030, 2, 256), (5, 32, 128)])
@pytest.mark.parametrize("half", [False, True], ids=["f32", "f16"])
def test_set_rows_bits(mx, t, n, H, D, half):
    """Codes and scales of the named rows are the definition's bits; the others keep theirs."""
    import torch
    rng = np.random.default_rng(n * D + H)
    x = (rng.standard_normal((n, H, D)) * 10.0 ** rng.uniform(-4, 3, (n, H, 1))).astype(np.float16 if half else np.float32)
    rows = n + 9
    c = noisy_cache(mx, t, rows, H, D)
    q0, d0 = cpu(c.q), cpu(c.d)
    at = rng.permutation(rows)[:n]
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    mx.set_rows([(c, gpu(x))], gpu(at.astype(np.int64 if n % 2 else np.int32)), err=err)
    codes, d = R.quantize(x, t)
    q0[at], d0[at] = codes, d
    assert np.array_equal(cpu(c.q), q0)
    assert np.array_equal(cpu(c.d).view(np.uint16), d0.view(np.uint16))
    assert int(err) == 0


def test_set_rows_several_caches_and_layouts(mx):
    """Four caches of all types in one call: token-major, head-major (a strided view), a slice of a
    longer cache, and rows without heads; plain rows strided too."""
    import torch
    n, H, D, rows = 45, 4, 64, 80
    rng = np.random.default_rng(3)
    wide = gpu(rng.standard_normal((n, H, 2 * D)).astype(np.float32))
    x = wide[:, :, D:]
    hm = noisy_cache(mx, Q4_0, H, rows, D).permute(1, 0, 2)
    sl = noisy_cache(mx, Q8_0, rows + 20, H, D)[7:7 + rows]
    f16 = mx.kv_cache(mx.F16, rows, H, D)
    flat = noisy_cache(mx, Q8_0, rows, H * D)
    at = rng.permutation(rows)[:n]
    mx.set_rows([(hm, x), (sl, x), (f16, x), (flat, x.reshape(n, H * D))], gpu(at))
    xn = cpu(x)
    for c, t in ((hm, Q4_0), (sl, Q8_0)):
        codes, d = R.quantize(xn, t)
        assert np.array_equal(cpu(c.q[gpu(at)]), codes) and np.array_equal(cpu(c.d[gpu(at)]).view(np.uint16), d.view(np.uint16))
    assert np.array_equal(cpu(f16.q[gpu(at)]), xn.astype(np.float16))
    codes, d = R.quantize(xn.reshape(n, -1), Q8_0)
    assert np.array_equal(cpu(flat.q[gpu(at)]), codes)
    got = mx.get_rows([hm, sl, f16], gpu(at))
    assert np.array_equal(cpu(got[0]), R.values(*R.quantize(xn, Q4_0), Q4_0).astype(np.float32))
    assert np.array_equal(cpu(got[1]), R.values(*R.quantize(xn, Q8_0), Q8_0).astype(np.float32))
    assert np.array_equal(cpu(got[2]), xn.astype(np.float16).astype(np.float32))
    whole = mx.get_rows([flat])[0]
    assert whole.shape == (rows, H * D) and np.array_equal(cpu(whole[gpu(at)]), R.values(codes, d, Q8_0).astype(np.float32))


@pytest.mark.parametrize("t", TYPES, ids=ids)
def test_set_rows_repeated_and_foreign_indices(mx, t):
    """Of rows with one index the last stays whole; indices outside the cache write nothing and set the flag."""
    import torch
    n, H, D, rows = 700, 2, 128, 40
    rng = np.random.default_rng(5)
    x = rng.standard_normal((n, H, D)).astype(np.float32)
    at = rng.integers(-3, rows + 3, n)
    at[n // 2:n // 2 + 9] = 17
    c = noisy_cache(mx, t, rows, H, D)
    q0, d0 = cpu(c.q), cpu(c.d)
    codes, d = R.quantize(x, t)
    for i, r in enumerate(at):
        if 0 <= r < rows:
            q0[r], d0[r] = codes[i], d[i]
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    for _ in range(3):
        mx.set_rows([(c, gpu(x))], gpu(at), err=err)
        assert np.array_equal(cpu(c.q), q0) and np.array_equal(cpu(c.d).view(np.uint16), d0.view(np.uint16))
    assert int(err) == 1
    out = torch.full((n, H, D), 7.0, device="cuda")
    err.zero_()
    mx.get_rows([c], gpu(at), out=[out], err=err)
    inside = (at >= 0) & (at < rows)
    got = cpu(out)
    assert int(err) == 1 and (got[~inside] == 7.0).all()
    assert np.array_equal(got[inside], R.values(q0, d0, t)[at[inside]].astype(np.float32))


@pytest.mark.parametrize("t", TYPES, ids=ids)
@pytest.mark.parametrize("wide", [False, True, None], ids=["int32", "int64", "all"])
def test_set_rows_of_a_whole_context(mx, t, wide):
    """More rows than one launch takes, into two caches, indices repeated near and far: the last row stays."""
    n, rows, H, D = 40000, 45000, 2, 32
    rng = np.random.default_rng(n)
    x, y = (rng.standard_normal((n, H, D)).astype(np.float32) for _ in range(2))
    at = np.arange(n) if wide is None else rng.integers(0, rows, n).astype(np.int64 if wide else np.int32)
    c, f = noisy_cache(mx, t, rows, H, D), mx.kv_cache(mx.F16, rows, H, D)
    q0, d0 = cpu(c.q).copy(), cpu(c.d).copy()
    mx.set_rows([(c, gpu(x)), (f, gpu(y))], None if wide is None else gpu(at))
    codes, d = R.quantize(x, t)
    q0[at], d0[at] = codes, d          # numpy assigns in order: the last one stays
    want = np.zeros((rows, H, D), np.float16)
    want[at] = y.astype(np.float16)
    assert np.array_equal(cpu(c.q), q0) and np.array_equal(cpu(c.d).view(np.uint16), d0.view(np.uint16))
    assert np.array_equal(cpu(f.q), want)


@pytest.mark.parametrize("t", TYPES, ids=ids)
def test_set_rows_special_blocks(mx, t):
    """Zeros, ties of both signs, halves between codes, magnitudes from f32's subnormals to past the
    scale's range, infinities and NaN, one kind a block."""
    x = np.zeros((16, 32), np.float32)
    rng = np.random.default_rng(9)
    x[1] = 2.5
    x[2, [3, 20]] = [-4.0, 4.0]
    x[3, [3, 20]] = [4.0, -4.0]
    x[4, [19, 5]] = [-4.0, 4.0]
    x[5] = np.arange(32) / 2 - 8
    x[6, :] = np.linspace(-127, 127, 32)
    x[6, 0] = 127
    x[7] = rng.standard_normal(32) * 1e-41
    x[8] = rng.standard_normal(32) * 1e-38
    x[9] = rng.standard_normal(32) * 1e-8
    x[10] = rng.standard_normal(32) * 1e5
    x[11] = rng.standard_normal(32) * 1e8          # the scale passes fp16: infinite, as ggml's
    x[12, 31] = np.inf
    x[13, 4] = -np.inf
    x[14, 17] = np.nan
    x[15] = -0.0
    c = noisy_cache(mx, t, 16, 32)
    mx.set_rows([(c, gpu(x))])
    codes, d = R.quantize(x, t)
    assert np.array_equal(cpu(c.q), codes)
    got = cpu(c.d)
    assert np.array_equal(np.isnan(got), np.isnan(d)) and np.array_equal(got[~np.isnan(d)].view(np.uint16), d[~np.isnan(d)].view(np.uint16))
    back = cpu(mx.get_rows([c])[0])
    assert np.isnan(back[12:15]).all() and np.isfinite(back[:11]).all()


# ---- GET_ROWS -------------------------------------------------------------------------------

@pytest.mark.parametrize("t", TYPES, ids=ids)
@pytest.mark.parametrize("n,H,D", [(1, 1, 32), (33, 8, 64), (257, 3, 160), (1000, 8, 128)])
def test_get_rows_values(mx, t, n, H, D):
    """F32 exact, F16 rounded once, with repeated indices, int32 and int64, and without."""
    import torch
    rng = np.random.default_rng(n)
    c = noisy_cache(mx, t, n, H, D, seed=n)
    want = R.values(cpu(c.q), cpu(c.d), t)
    at = rng.integers(0, n, 2 * n)
    for idx in (at.astype(np.int32), at.astype(np.int64)):
        assert np.array_equal(cpu(mx.get_rows([c], gpu(idx))[0]), want[at].astype(np.float32))
    got = cpu(mx.get_rows([c], None, torch.float16)[0])
    assert np.array_equal(got, want.astype(np.float32).astype(np.float16))


def test_rows_of_nothing(mx):
    """n = 0 returns without a launch and without touching the cache."""
    import torch
    c = noisy_cache(mx, Q8_0, 4, 2, 64)
    q0 = cpu(c.q)
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    mx.set_rows([(c, torch.empty(0, 2, 64, device="cuda"))], none)
    assert mx.get_rows([c], none)[0].shape == (0, 2, 64)
    assert np.array_equal(cpu(c.q), q0)


def test_rows_past_32_bit_offsets(mx):
    """A cache whose last rows lie past 2^31 elements (and 2^32 bytes of plain values are not needed)."""
    H, D = 8, 256
    rows = (1 << 31) // (H * D) + 77
    c = mx.kv_cache(Q4_0, rows, H, D)
    rng = np.random.default_rng(1)
    x = rng.standard_normal((3, H, D)).astype(np.float32)
    at = np.array([rows - 1, 5, (1 << 31) // (H * D) + 3])
    mx.set_rows([(c, gpu(x))], gpu(at))
    codes, d = R.quantize(x, Q4_0)
    assert np.array_equal(cpu(c.q[gpu(at)]), codes)
    assert np.array_equal(cpu(mx.get_rows([c], gpu(at))[0]), R.values(codes, d, Q4_0).astype(np.float32))


# ---- FLASH_ATTN_EXT -------------------------------------------------------------------------

def causal(T, KV, lens=None):
    """[S][T][KV rounded up to 8] fp16: the last query of a sequence sees its whole length."""
    lens = [KV] if lens is None else lens
    j, t = np.arange((KV + 7) // 8 * 8)[None, None, :], np.arange(T)[None, :, None]
    return np.where(j > np.array(lens)[:, None, None] - T + t, -np.inf, 0.0).astype(np.float16)


def attn_case(mx, kt, vt, S, T, H, HK, KV, D, DV, seed=0, head_major=False, q_half=False, scale_up=1.0):
    rng = np.random.default_rng(seed + 1000 * T + KV + D)
    q = (rng.standard_normal((S, H, T, D)) * scale_up).astype(np.float16 if q_half else np.float32)
    kq, kd = R.quantize(rng.standard_normal((S, KV, HK, D)), kt)
    vq, vd = R.quantize(rng.standard_normal((S, KV, HK, DV)), vt)
    kn, vn = R.values(kq, kd, kt).transpose(0, 2, 1, 3), R.values(vq, vd, vt).transpose(0, 2, 1, 3)
    if head_major:
        kc, vc = (mx.KvCache(t, gpu(c.transpose(0, 2, 1, 3)), gpu(d.transpose(0, 2, 1, 3))) for t, c, d in ((kt, kq, kd), (vt, vq, vd)))
    else:
        kc, vc = (mx.KvCache(t, gpu(c), gpu(d)).permute(0, 2, 1, 3) for t, c, d in ((kt, kq, kd), (vt, vq, vd)))
    return q, kn, vn, kc, vc


def check(got, q, kn, vn, mask, scale, softcap=0.0, half_out=False, what=""):
    for s in range(q.shape[0]):
        m = None if mask is None else mask[s if mask.shape[0] > 1 else 0].astype(np.float64)
        want, tol = R.attention(q[s].astype(np.float64), kn[s], vn[s], m, scale, softcap)
        if half_out:
            tol = tol + np.abs(want) * R.HALF + 2.0 ** -25
        d = np.abs(got[s].astype(np.float64) - want)
        assert np.isfinite(got[s]).all() and (d <= tol).all(), (what, s, float((d - tol).max()), float(d.max()))


@pytest.mark.parametrize("types", MIXES, ids=ids)
@pytest.mark.parametrize("T,KV", [(1, 1), (1, 2), (1, 33), (1, 777), (3, 64), (7, 1000), (16, 129), (33, 500), (70, 389)])
def test_attention_lengths(mx, form, types, T, KV):
    """From one token on one key to ragged prompts, GQA of four, causal."""
    H, HK, D = 8, 2, 128
    q, kn, vn, kc, vc = attn_case(mx, *types, 1, T, H, HK, KV, D, D)
    m = causal(T, KV)
    for ns in (0, 1, 3):
        got = cpu(mx.flash_attn_q(gpu(q), kc, vc, gpu(m), D ** -0.5, nsplit=ns))
        check(got, q, kn, vn, m, D ** -0.5, what=ns)


@pytest.mark.parametrize("types", MIXES, ids=ids)
@pytest.mark.parametrize("D,DV,H,HK", [(32, 32, 4, 4), (64, 64, 6, 3), (96, 96, 5, 1), (128, 64, 8, 2), (160, 96, 4, 2), (192, 128, 16, 2),
                                       (256, 256, 8, 4), (224, 160, 9, 3)])
@pytest.mark.parametrize("T", [1, 5, 40])
def test_attention_head_dims(mx, form, types, D, DV, H, HK, T):
    """Head dims that are multiples of 32, groups from 1 to 8 and odd ones, a soft-cap, no mask."""
    KV, cap = 203, 10.0
    q, kn, vn, kc, vc = attn_case(mx, *types, 1, T, H, HK, KV, D, DV, head_major=T == 5)
    got = cpu(mx.flash_attn_q(gpu(q), kc, vc, None, D ** -0.5, softcap=cap))
    check(got, q, kn, vn, None, D ** -0.5, cap)


@pytest.mark.parametrize("types", [MIXES[0], MIXES[2]], ids=ids)
@pytest.mark.parametrize("T,half", [(1, False), (1, True), (6, True), (40, True)])
def test_attention_streams(mx, form, types, T, half):
    """Five sequences of different lengths (one of them empty), fp16 queries and outputs, outputs with a
    wider row stride left alone beside it."""
    import torch
    S, H, HK, D, KV = 5, 8, 2, 64, 300
    lens = [300, 17, 0, 133, 64]
    q, kn, vn, kc, vc = attn_case(mx, *types, S, T, H, HK, KV, D, D, q_half=half)
    m = causal(T, KV, lens)
    wide = torch.full((S, T, H, D + 8), float("nan"), dtype=torch.float16 if half else torch.float32, device="cuda")
    mx.flash_attn_q(gpu(q), kc, vc, gpu(m), 0.125, out=wide[..., :D])
    w = cpu(wide)
    assert np.isnan(w[..., D:]).all()
    check(w[..., :D], q, kn, vn, m, 0.125, half_out=half)
    assert (w[2, ..., :D] == 0).all()
    one = cpu(mx.flash_attn_q(gpu(q), kc, vc, gpu(m[:1]), 0.125))        # one mask for all of them
    check(one, q, kn, vn, m[:1], 0.125)


@pytest.mark.parametrize("types", MIXES, ids=ids)
@pytest.mark.parametrize("D,DV,G,T", [(64, 64, 4, 11), (96, 96, 1, 47), (128, 128, 4, 12), (192, 128, 4, 9), (224, 224, 4, 9)])
def test_attention_many_short_sequences(mx, form, types, D, DV, G, T):
    """More row tiles than compute units (24 sequences x 4 heads x 3 tiles of 16), an odd number of them a
    head, each sequence at its own length, scattered hidden keys and whole hidden tiles, one empty row."""
    S, HK, KV = 24, 4, 170
    rng = np.random.default_rng(D)
    q, kn, vn, kc, vc = attn_case(mx, *types, S, T, G * HK, HK, KV, D, DV)
    m = causal(T, KV, [1 + (37 * s) % KV for s in range(S)])
    m[rng.random(m.shape) > 0.8] = -np.inf
    m[:, 4:, 64:96] = -np.inf
    m[5, 2, :] = -np.inf
    for ns in (0, 2):
        got = cpu(mx.flash_attn_q(gpu(q), kc, vc, gpu(m), D ** -0.5, nsplit=ns))
        check(got, q, kn, vn, m, D ** -0.5, what=ns)
        assert (got[5, 2] == 0).all()


@pytest.mark.parametrize("types", MIXES, ids=ids)
@pytest.mark.parametrize("T", [1, 9, 64])
def test_attention_mask_holes(mx, form, types, T):
    """Scattered hidden keys, whole hidden tiles, rows that see nothing, masks of fp16's lowest value,
    biases; what the cache holds under a mask that hides it from every query (NaN and infinite
    scales, all codes) does not matter."""
    H, HK, D, KV = 8, 2, 128, 640
    q, kn, vn, kc, vc = attn_case(mx, *types, 1, T, H, HK, KV, D, D, seed=4)
    rng = np.random.default_rng(T)
    m = np.zeros((1, T, KV), np.float16)
    m[rng.random((1, T, KV)) > 0.6] = -np.inf
    m[0, :, 100:230] = -np.inf
    m[0, :, 600:] = -np.inf
    m[rng.random((1, T, KV)) > 0.95] += np.float16(-1.5)
    if T > 1:
        m[0, 3, :] = -np.inf
        m[0, 5, :] = -65504.0          # every key as low as fp16 goes: all alike, not hidden
        m[0, 5, 100:230] = m[0, 5, 600:] = -np.inf
    hidden = (m[0] == -np.inf).all(0)
    assert hidden[100:230].all()
    h = np.flatnonzero(hidden)
    for c in (kc, vc):
        for i, bad in enumerate((float("nan"), INF, -INF)):
            c.d[0][:, gpu(h[i::5])] = bad
    for ns in (0, 1, 2):
        got = cpu(mx.flash_attn_q(gpu(q), kc, vc, gpu(m), D ** -0.5, nsplit=ns))
        check(got, q, kn, vn, m, D ** -0.5, what=ns)
        if T > 1:
            assert (got[0, 3] == 0).all()


@pytest.mark.parametrize("T", [1, 9, 64])
@pytest.mark.parametrize("plane", ["k", "v"])
def test_attention_nan_reaches_who_sees_it(mx, form, T, plane):
    """A visible key whose scale is NaN makes the rows of the queries that see it NaN, and no others."""
    H, HK, D, KV = 4, 2, 64, 200
    q, kn, vn, kc, vc = attn_case(mx, Q8_0, Q4_0, 1, T, H, HK, KV, D, D, seed=8)
    m = np.zeros((1, T, KV), np.float16)
    m[0, 1::2, 70] = -np.inf
    (kc if plane == "k" else vc).d[0, 0, 70, 1] = float("nan")
    if T == 1:      # alone: the only key of a row
        m[0, 0, :] = -np.inf
        m[0, 0, 70] = 0
    for ns in (0, 1, 2):
        got = cpu(mx.flash_attn_q(gpu(q), kc, vc, gpu(m), 0.125, nsplit=ns))
        assert np.isnan(got[0, 0::2, :2]).all() and np.isfinite(got[0, 1::2]).all() and np.isfinite(got[0, :, 2:]).all(), ns
        check(got[:, 1::2], q[:, :, 1::2], kn, vn, m[:, 1::2], 0.125)


@pytest.mark.parametrize("types", [MIXES[0], MIXES[1]], ids=ids)
@pytest.mark.parametrize("T", [1, 40])
def test_attention_ranges(mx, form, types, T):
    """Scores past fp16 (one key wins by far), queries whose scaled values pass fp16, caches of tiny
    and of large values, and blocks of very different scales."""
    H, HK, D, KV = 4, 2, 64, 300
    for up, ks, vs in ((1e6, 1.0, 1.0), (1.0, 1e-3, 1e-2), (0.02, 300.0, 3000.0)):
        rng = np.random.default_rng(int(up) + T)
        q = (rng.standard_normal((1, H, T, D)) * up).astype(np.float32)
        spread = 10.0 ** rng.uniform(-1, 1, (1, KV, HK, 1))
        kq, kd = R.quantize(rng.standard_normal((1, KV, HK, D)) * ks, types[0])
        vq, vd = R.quantize(rng.standard_normal((1, KV, HK, D)) * vs * spread, types[1])
        kn, vn = R.held(kq, kd, types[0]).transpose(0, 2, 1, 3), R.held(vq, vd, types[1]).transpose(0, 2, 1, 3)
        kc, vc = (mx.KvCache(t, gpu(c), gpu(d)).permute(0, 2, 1, 3) for t, c, d in ((types[0], kq, kd), (types[1], vq, vd)))
        got = cpu(mx.flash_attn_q(gpu(q), kc, vc, None, 0.125))
        assert np.isfinite(got).all()
        # below 2^-14 an fp16 V is off by at most 2^-25 instead
        want, tol = R.attention(q[0], kn[0], vn[0], None, 0.125)
        assert (np.abs(got[0] - want) <= tol + 2.0 ** -25).all(), (up, float((np.abs(got[0] - want) - tol).max()))


@pytest.mark.parametrize("KV,heads", [(300, 1 << 16), (150, 1 << 17)])
def test_attention_past_32_bit_offsets(mx, form, KV, heads):
    """A cache whose keys lie 2^23 and 2^24 elements apart, past 2^31 of them in all, two of its heads in use."""
    H, HK, D, T = 4, 2, 128, 3
    rng = np.random.default_rng(KV)
    q = rng.standard_normal((1, H, T, D)).astype(np.float32)
    x, y = (rng.standard_normal((KV, HK, D)).astype(np.float32) for _ in range(2))
    whole = mx.kv_cache(Q4_0, KV, heads, D)
    k, v = whole[:, heads - 3:heads - 1], whole[:, 7:9]
    mx.set_rows([(k, gpu(x)), (v, gpu(y))])
    m = causal(T, KV)
    kn, vn = (R.values(*R.quantize(p, Q4_0), Q4_0).transpose(1, 0, 2)[None] for p in (x, y))
    got = cpu(mx.flash_attn_q(gpu(q[0]), k.permute(1, 0, 2), v.permute(1, 0, 2), gpu(m[0]), D ** -0.5))
    check(got[None], q, kn, vn, m, D ** -0.5)


def test_attention_no_keys(mx, form):
    """KV = 0: zeros."""
    import torch
    kc, vc = mx.kv_cache(Q8_0, 2, 8, 64)[:, :0], mx.kv_cache(Q4_0, 2, 8, 64)[:, :0]
    for T in (1, 40):
        got = mx.flash_attn_q(torch.randn(4, T, 64, device="cuda"), kc, vc, None, 0.125)
        assert (cpu(got) == 0).all()


def test_attention_same_bits_and_same_as_a_decoded_cache(mx, form):
    """Two calls give equal bits; the fp16 attention on the cache read back as fp16 agrees."""
    import torch
    H, HK, D = 8, 2, 128
    for T, KV in ((1, 2000), (12, 2000), (200, 1024)):
        q, kn, vn, kc, vc = attn_case(mx, Q8_0, Q4_0, 1, T, H, HK, KV, D, D)
        m = gpu(causal(T, KV))
        a, b = (mx.flash_attn_q(gpu(q), kc, vc, m, D ** -0.5) for _ in range(2))
        assert torch.equal(a, b)
        k16, v16 = (gpu(x.astype(np.float32).astype(np.float16)[0]) for x in (kn, vn))
        ref = mx.flash_attn(gpu(q)[0], k16, v16, m[0], D ** -0.5)
        # both within the same bound of the exact result; the scores are O(1) here
        assert float((a[0] - ref).abs().max()) <= 4e-3


# ---- together -------------------------------------------------------------------------------

@pytest.mark.parametrize("T,KV", [(1, 3000), (40, 700)])
def test_attention_on_two_streams_at_once(mx, form, T, KV):
    """Two calls in flight with a workspace each give the bits of one after the other."""
    import torch
    H, HK, D = 8, 2, 64
    cases = [attn_case(mx, Q4_0, Q8_0, 1, T, H, HK, KV - 9 * i, D, D, seed=i) for i in range(2)]
    masks = [gpu(causal(T, KV - 9 * i)) for i in range(2)]
    qs = [gpu(c[0]) for c in cases]
    alone = [cpu(mx.flash_attn_q(q, c[3], c[4], m, 0.125)) for q, c, m in zip(qs, cases, masks)]
    outs = [torch.empty(1, T, H, D, device="cuda") for _ in range(2)]
    spaces = [torch.empty(mx.flash_attn_q_workspace(q, c[3], c[4], m, o), dtype=torch.uint8, device="cuda")
              for q, c, m, o in zip(qs, cases, masks, outs)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for st, q, c, m, o, w in zip(streams, qs, cases, masks, outs, spaces):
            with torch.cuda.stream(st):
                mx.flash_attn_q(q, c[3], c[4], m, 0.125, out=o, workspace=w)
    torch.cuda.synchronize()
    for o, a in zip(outs, alone):
        assert np.array_equal(cpu(o), a)


def test_decode_loop_on_another_stream_and_in_a_graph(mx, form):
    """A sequence grown as it would be: a prompt stored and attended to, then token by token, on a
    stream of its own; the last token's step captured into a graph and replayed with new inputs and
    eager work in between, each replay equal to the eager step."""
    import torch
    H, HK, D, ctx, T0 = 8, 2, 64, 128, 50
    rng = np.random.default_rng(2)
    kc, vc = mx.kv_cache(Q8_0, ctx, HK, D), mx.kv_cache(Q4_0, ctx, HK, D)
    kv = kc.permute(1, 0, 2), vc.permute(1, 0, 2)
    K, V = (rng.standard_normal((ctx, HK, D)).astype(np.float32) for _ in range(2))
    Q = rng.standard_normal((H, ctx, D)).astype(np.float32)
    kn, vn = R.values(*R.quantize(K, Q8_0), Q8_0).transpose(1, 0, 2), R.values(*R.quantize(V, Q4_0), Q4_0).transpose(1, 0, 2)
    full = np.where(np.arange(ctx)[None, :] > np.arange(ctx)[:, None], -np.inf, 0.0).astype(np.float16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        steps = [(0, T0)] + [(i, i + 1) for i in range(T0, T0 + 8)]
        for a, b in steps:
            mx.set_rows([(kc, gpu(K[a:b])), (vc, gpu(V[a:b]))], torch.arange(a, b, device="cuda"))
            got = mx.flash_attn_q(gpu(Q[:, a:b]), *kv, gpu(full[a:b]), 0.125)
            side.synchronize()
            want, tol = R.attention(Q[:, a:b], kn, vn, full[a:b], 0.125)
            assert (np.abs(got.cpu().numpy() - want) <= tol).all(), a
        # one step as a graph: its inputs are copied into fixed buffers
        xk, xv = (torch.zeros(1, HK, D, device="cuda") for _ in range(2))
        q, m = torch.zeros(H, 1, D, device="cuda"), torch.zeros(1, ctx, dtype=torch.float16, device="cuda")
        at, out = torch.zeros(1, dtype=torch.int64, device="cuda"), torch.zeros(1, H, D, device="cuda")
        ws = torch.empty(mx.flash_attn_q_workspace(q, *kv, m, out), dtype=torch.uint8, device="cuda")
        ws.random_(0, 256)

        def step():
            mx.set_rows([(kc, xk), (vc, xv)], at)
            mx.flash_attn_q(q, *kv, m, 0.125, out=out, workspace=ws)
        for dst, src in ((xk, K[:1]), (xv, V[:1]), (q, Q[:, :1]), (m, full[:1])):
            dst.copy_(gpu(src))
        step()
        side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    with torch.cuda.stream(side):
        for i in range(T0 + 8, T0 + 13):
            for dst, src in ((xk, K[i:i + 1]), (xv, V[i:i + 1]), (q, Q[:, i:i + 1]), (m, full[i:i + 1])):
                dst.copy_(gpu(src))
            at.fill_(i)
            graph.replay()
            side.synchronize()
            got = out.clone()
            ws.random_(0, 256)               # nothing is kept in the workspace between calls
            step()                            # the eager step on the same inputs
            side.synchronize()
            assert torch.equal(got, out)
            want, tol = R.attention(Q[:, i:i + 1], kn, vn, full[i:i + 1], 0.125)
            assert (np.abs(got.cpu().numpy() - want) <= tol).all(), i

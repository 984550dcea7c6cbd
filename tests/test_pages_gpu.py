"""A KV cache in pages on the GPU against plain numpy (pages_oracle): stored bits and rotated queries equal to the
definition's, attention of chains and trees within the bound that fp16 operands allow, kept rows bit by bit; numbers
that a caller should not pass; the three as a decoding loop uses them, eager and captured."""
import numpy as np
import pytest

import kv_norm
import kv_oracle as R
import pages_oracle as P

pytestmark = pytest.mark.gpu

F16, Q4_0, Q8_0 = P.F16, R.Q4_0, R.Q8_0
NAME = {Q8_0: "q8_0", Q4_0: "q4_0", F16: "f16"}
MIXES = [(Q8_0, Q8_0), (Q4_0, Q4_0), (Q8_0, Q4_0), (Q4_0, Q8_0)]
ATTENDED = MIXES + [(F16, F16)]


def ids(v):
    return NAME.get(v) if isinstance(v, int) else "-".join(str(NAME.get(t, t)) for t in v) if isinstance(v, tuple) else None


@pytest.fixture(scope="module")
def mx(torch_cuda):
    import ggml_mi355x
    ggml_mi355x.lib()
    return ggml_mi355x


@pytest.fixture(params=["1 16", "1 32", "0 ", " "], ids=["direct", "direct32", "decoded", "chosen"])
def form(request, monkeypatch):
    """Attention under every form (16 and 32 rows a wave; chains over a quantized cache decoded first) and the library's choice."""
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


def i32(a):
    return gpu(np.asarray(a, np.int32))


def cache_of(mx, t, rows, H, D, rng, junk=0.0):
    """A cache of N(0, 1) values and its planes; a share `junk` of the rows holds NaN (scales, F16 values) instead."""
    import torch
    pl = P.planes(rng.standard_normal((rows, H, D)).astype(np.float32), t)
    bad = rng.random(rows) < junk
    pl[-1][bad] = 0x7E00
    if t == F16:
        return mx.KvCache(F16, gpu(pl[0].view(np.float16))), pl
    return mx.KvCache(t, gpu(pl[0]), gpu(pl[1].view(np.float16))), pl


def planes_of(c):
    return [cpu(c.q).view(np.uint16)] if c.type == F16 else [cpu(c.q), cpu(c.d).view(np.uint16)]


def same(a, b):
    return len(a) == len(b) and all(np.array_equal(x, y) for x, y in zip(a, b))


def tables(rng, past, new, page, spare=3, extra=1):
    """(table, pages): every sequence's own pages in no order; entries behind its last are no page's number."""
    used = [(p + n + page - 1) // page for p, n in zip(past, new)]
    pages = sum(used) + spare
    order = rng.permutation(pages)
    table = np.full((len(past), max(used) + extra), -7, np.int32)
    at = 0
    for s, n in enumerate(used):
        table[s, :n] = order[at:at + n]
        at += n
    return table, pages


def tree(rng, S, T):
    return np.stack([[int(rng.integers(-1, t)) if t else -1 for t in range(T)] for _ in range(S)]).astype(np.int32)


def zeros_i32():
    import torch
    return torch.zeros(1, dtype=torch.int32, device="cuda")


# ---- append ---------------------------------------------------------------------------------

APPEND = [  # S, T, tree, past, page, H, HK, D, DV, n_rot, neox, source f16
    (1, 1, False, [5], 32, 4, 2, 64, 64, 64, True, False),
    (1, 1, False, [0], 64, 32, 8, 128, 128, 128, False, True),
    (3, 5, False, [31, 0, 1000], 32, 3, 3, 96, 96, 48, True, False),
    (2, 64, True, [63, 130000], 96, 8, 2, 128, 128, 64, False, False),
    (5, 17, True, [1, 2, 33, 300, 95], 32, 4, 4, 192, 128, 192, True, True),
    (1, 700, False, [100], 128, 2, 1, 256, 256, 256, True, False),
    (1, 300, False, [0], 256, 2, 2, 32, 64, 8, False, True),
    (2, 9, False, [7, 8], 64, 0, 2, 64, 32, 24, True, True),
    (2, 3, True, [7, 8], 64, 2, 2, 64, 32, 0, False, False),
]


@pytest.mark.parametrize("kt,vt", ATTENDED + [(F16, Q8_0)], ids=lambda t: NAME[t])
@pytest.mark.parametrize("case", APPEND, ids=lambda c: "S%dT%d%sD%dr%d" % (c[0], c[1], "t" if c[2] else "c", c[7], c[9]))
def test_append_bits(mx, kt, vt, case):
    """Rows of the real tokens hold the definition's bits, all others keep theirs; so do queries."""
    import torch
    S, T, is_tree, past, page, H, HK, D, DV, n_rot, neox, half = case
    rng = np.random.default_rng(S * 1000 + T + D)
    new = [T] if S == 1 else [int(n) for n in rng.integers(0, T + 1, S)]
    if S > 1:
        new[0] = T
    table, pages = tables(rng, past, new, page)
    rows = pages * page + 5
    kc, kp = cache_of(mx, kt, rows, HK, D, rng)
    vc, vp = cache_of(mx, vt, rows, HK, DV, rng)
    dt = np.float16 if half else np.float32
    k, v, q = (rng.standard_normal(s).astype(dt) for s in ((S, T, HK, D), (S, T, HK, DV), (S, T, max(H, 1), D)))
    parents = tree(rng, S, T) if is_tree else None
    freq = (10000.0 ** (-np.arange(n_rot // 2) / max(1, n_rot // 2))).astype(np.float32)
    step = mx.KvStep(i32(table), i32(past), T, page, n_new=i32(new), parents=None if parents is None else i32(parents))
    rope = mx.Rope(gpu(freq), neox=neox, mscale=1.125 if T == 17 else 1.0) if n_rot else None
    err, q_out = zeros_i32(), torch.full((S, T, max(H, 1), D), 7.0, device="cuda", dtype=torch.float32)
    got = mx.kv_append(step, kc, vc, gpu(k), gpu(v), rope=rope, q=gpu(q) if H else None, q_out=q_out if H else None, err=err)
    assert (got is q_out) == (H > 0)
    want_q = np.full(q.shape, 7.0, np.float32)
    for s in range(S):
        if not new[s]:
            continue
        pos = [past[s] + len(w) - 1 for w in P.ways(None if parents is None else parents[s], new[s])]
        at = [P.row(table[s], page, past[s] + t) for t in range(new[s])]
        m = 1.125 if T == 17 else 1.0
        for p, x in zip(kp, P.planes(P.rotate(k[s, :new[s]], pos, freq, neox, m), kt)):
            p[at] = x
        for p, x in zip(vp, P.planes(v[s, :new[s]].astype(np.float32), vt)):
            p[at] = x
        want_q[s, :new[s]] = P.rotate(q[s, :new[s]], pos, freq, neox, m)
    assert same(planes_of(kc), kp) and same(planes_of(vc), vp)
    assert not H or np.array_equal(cpu(q_out), want_q)
    assert int(err) == 0


def test_append_strided_positions_and_f16_queries(mx):
    """Sources and queries as slices of one projection, an fp16 result in place, given positions, a head-major cache."""
    import torch
    S, T, H, HK, D, page = 2, 6, 4, 2, 64, 32
    rng = np.random.default_rng(4)
    past, new = [40, 3], [6, 5]
    table, pages = tables(rng, past, new, page)
    rows = pages * page
    base = mx.kv_cache(mx.Q8_0, HK, rows, D)
    kc, vc = base.permute(1, 0, 2), mx.kv_cache(mx.F16, rows, HK, D)
    x = rng.standard_normal((S, T, (H + 2 * HK) * D)).astype(np.float16)
    qkv = gpu(x).reshape(S, T, H + 2 * HK, D)
    q, k, v = qkv[:, :, :H], qkv[:, :, H:H + HK], qkv[:, :, H + HK:]
    pos = rng.integers(0, 1 << 20, (S, T)).astype(np.int32)
    wide = gpu(np.concatenate([pos, pos], 1))[:, :T]
    freq = mx.rope_freqs(D, 500000.0)
    step = mx.KvStep(i32(np.concatenate([table, table], 1))[:, :table.shape[1]], i32(past), T, page, n_new=i32(new))
    mx.kv_append(step, kc, vc, k, v, rope=mx.Rope(freq, neox=False, positions=wide), q=q, q_out=q)
    xs = x.reshape(S, T, H + 2 * HK, D)
    got, gk, gv = cpu(qkv), planes_of(kc), planes_of(vc)
    for s in range(S):
        n = new[s]
        at = [P.row(table[s], page, past[s] + t) for t in range(n)]
        turned = P.rotate(xs[s, :n], pos[s, :n], cpu(freq), False)
        assert np.array_equal(got[s, :n, :H], turned[:, :H].astype(np.float16)) and np.array_equal(got[s, n:], xs[s, n:])
        assert np.array_equal(got[s, :, H:], xs[s, :, H:])
        assert same([p[at] for p in gk], P.planes(turned[:, H:H + HK], Q8_0))
        assert same([p[at] for p in gv], P.planes(xs[s, :n, H + HK:].astype(np.float32), F16))


@pytest.mark.parametrize("neox", [False, True])
def test_append_far_positions(mx, neox):
    """Angles of any int32 position, to the last bit of the rotated values."""
    import torch
    S, T, H, HK, D, page = 1, 600, 2, 1, 64, 64
    rng = np.random.default_rng(12)
    table, pages = tables(rng, [0], [T], page)
    kc, kp = cache_of(mx, F16, pages * page, HK, D, rng)
    vc, vp = cache_of(mx, Q8_0, pages * page, HK, D, rng)
    q, k, v = (rng.standard_normal((S, T, h, D)).astype(np.float32) for h in (H, HK, HK))
    pos = rng.integers(-2 ** 31, 2 ** 31, (S, T)).astype(np.int32)
    pos[0, :8] = [0, -1, 1, 2 ** 31 - 1, -2 ** 31, 355, 710, 52174]     # 355 and 710: next to multiples of pi
    freq = np.concatenate([[1.0, 3.75, 0.0, -0.5], 500000.0 ** (-np.arange(28) / 28)]).astype(np.float32)
    q_out = torch.empty(S, T, H, D, device="cuda")
    step = mx.KvStep(i32(table), i32([0]), T, page)
    mx.kv_append(step, kc, vc, gpu(k), gpu(v), rope=mx.Rope(gpu(freq), neox=neox, positions=gpu(pos)), q=gpu(q), q_out=q_out)
    at = [P.row(table[0], page, t) for t in range(T)]
    kp[0][at] = P.planes(P.rotate(k[0], pos[0], freq, neox), F16)[0]
    assert np.array_equal(cpu(q_out)[0], P.rotate(q[0], pos[0], freq, neox)) and same(planes_of(kc), kp)


@pytest.mark.parametrize("T,page", [(1, 32), (40, 32), (300, 64)])
def test_append_rows_that_two_tokens_share(mx, T, page):
    """Tables that share pages: of the tokens with one row the last, by sequence and number, stays whole."""
    S, HK, D = 6, 2, 128
    rng = np.random.default_rng(T)
    past = [int(n) for n in rng.integers(0, 70, S)]
    new = [int(n) for n in rng.integers(1, T + 1, S)]
    n_table = (70 + T + page - 1) // page + 1
    pages = max(3, n_table - 2)
    table = rng.integers(0, pages, (S, n_table)).astype(np.int32)
    kc, kp = cache_of(mx, Q8_0, pages * page, HK, D, rng)
    vc, vp = cache_of(mx, Q4_0, pages * page, HK, D, rng)
    k, v = (rng.standard_normal((S, T, HK, D)).astype(np.float32) for _ in range(2))
    step = mx.KvStep(i32(table), i32(past), T, page, n_new=i32(new))
    for _ in range(3):
        mx.kv_append(step, kc, vc, gpu(k), gpu(v))
    for s in range(S):
        for t in range(new[s]):
            r = P.row(table[s], page, past[s] + t)
            for pl, x, ty in ((kp, k, Q8_0), (vp, v, Q4_0)):
                for p, y in zip(pl, P.planes(x[s, t:t + 1], ty)):
                    p[r] = y[0]
    assert same(planes_of(kc), kp) and same(planes_of(vc), vp)


def test_append_shared_rows_of_nodes_without_a_way_up(mx):
    """A node that counts as padding writes no row, so an earlier token's that shares the row stays."""
    S, T, HK, D, page = 3, 12, 2, 64, 32
    rng = np.random.default_rng(31)
    past, new = [20, 20, 17], [12, 12, 9]
    table = np.array([[0, 1], [0, 1], [0, 2]], np.int32)
    parents = tree(rng, S, T)
    parents[1, 3], parents[1, 5], parents[1, 7] = 3, 5, 11
    parents[2, 1], parents[2, 4] = -5, 4
    parents[2, 6] = 4                                # below one that has no way up itself
    kc, kp = cache_of(mx, Q8_0, 3 * page, HK, D, rng)
    vc, vp = cache_of(mx, F16, 3 * page, HK, D, rng)
    k, v = (rng.standard_normal((S, T, HK, D)).astype(np.float32) for _ in range(2))
    err = zeros_i32()
    mx.kv_append(mx.KvStep(i32(table), i32(past), T, page, n_new=i32(new), parents=i32(parents)), kc, vc, gpu(k), gpu(v), err=err)
    for s in range(S):
        for t, w in enumerate(P.ways(parents[s], new[s])):
            if w is None:
                continue
            r = P.row(table[s], page, past[s] + t)
            for pl, x, ty in ((kp, k, Q8_0), (vp, v, F16)):
                for p, y in zip(pl, P.planes(x[s, t:t + 1], ty)):
                    p[r] = y[0]
    assert same(planes_of(kc), kp) and same(planes_of(vc), vp) and int(err) == 1


@pytest.mark.parametrize("S,T,page", [(2300, 1, 32), (1, 70000, 32), (2, 66000, 96)])
def test_append_in_several_launches(mx, S, T, page):
    """More sequences and tokens than a launch takes, and rows shared between those of different launches."""
    HK, D = 1, 32
    rng = np.random.default_rng(S + T)
    past = [int(n) for n in rng.integers(0, 50, S)]
    new = [T - int(n) for n in rng.integers(0, 2, S)]
    n_table = (50 + T) // page + 2
    pages = max(4, S * n_table * 2 // 3)
    table = rng.integers(0, pages, (S, n_table)).astype(np.int32)
    kc, kp = cache_of(mx, Q8_0, pages * page, HK, D, rng)
    vc, vp = cache_of(mx, F16, pages * page, HK, D, rng)
    q, k, v = (rng.standard_normal((S, T, HK, D)).astype(np.float32) for _ in range(3))
    freq = np.array([1.0, 0.1, 0.01, 0.001], np.float32)
    step = mx.KvStep(i32(table), i32(past), T, page, n_new=i32(new))
    got = cpu(mx.kv_append(step, kc, vc, gpu(k), gpu(v), rope=mx.Rope(gpu(freq)), q=gpu(q)))
    for s in range(S):
        n = new[s]
        if not n:
            continue
        j = past[s] + np.arange(n)
        at = table[s][j // page].astype(np.int64) * page + j % page
        turned = P.rotate(np.concatenate([k[s, :n], q[s, :n]], 1), j, freq, False)
        assert np.array_equal(got[s, :n], turned[:, 1:])
        last = np.unique(at[::-1], return_index=True)     # of the tokens with one row the last
        for pl, x, ty in ((kp, turned[:, :1], Q8_0), (vp, v[s, :n], F16)):
            for p, y in zip(pl, P.planes(x, ty)):
                p[last[0]] = y[::-1][last[1]]
    assert same(planes_of(kc), kp) and same(planes_of(vc), vp)


FAULTS = {   # past, new, what is done to the table; the tokens stored nevertheless
    "past_negative": ([-1, 4], [2, 2], None, {1: [0, 1]}),
    "past_behind": ([97, 4], [1, 2], None, {1: [0, 1]}),
    "new_negative": ([4, 4], [-3, 2], None, {1: [0, 1]}),
    "new_above": ([4, 4], [9, 2], None, {0: [0, 1, 2, 3], 1: [0, 1]}),
    "table_ends": ([94, 4], [4, 2], None, {0: [0, 1], 1: [0, 1]}),
    "page_negative": ([30, 4], [4, 2], (0, 1, -1), {0: [0, 1], 1: [0, 1]}),
    "page_above": ([30, 4], [4, 2], (0, 1, 7), {0: [0, 1], 1: [0, 1]}),
    "page_huge": ([30, 4], [4, 2], (0, 0, 2 ** 31 - 1), {0: [2, 3], 1: [0, 1]}),
    "past_huge": ([2 ** 31 - 1, 4], [4, 2], None, {1: [0, 1]}),
}


@pytest.mark.parametrize("name", FAULTS)
def test_append_numbers_out_of_range(mx, name):
    """Nothing but the rows that exist is written, and the flag is set; the other sequence is as ever."""
    import torch
    past, new, change, stored = FAULTS[name]
    T, page, HK, D = 4, 32, 1, 64
    rng = np.random.default_rng(8)
    table = np.array([[0, 1, 2], [3, 4, 5]], np.int32)
    if change:
        table[change[0], change[1]] = change[2]
    kc, kp = cache_of(mx, Q8_0, 7 * page + 31, HK, D, rng)
    vc, vp = cache_of(mx, F16, 7 * page + 40, HK, D, rng)
    k, v = (rng.standard_normal((2, T, HK, D)).astype(np.float32) for _ in range(2))
    step = mx.KvStep(i32(table), i32(past), T, page, n_new=i32(new))
    err = zeros_i32()
    mx.kv_append(step, kc, vc, gpu(k), gpu(v), q=gpu(k), err=err)
    for s, ts in stored.items():
        for t in ts:
            r = P.row(table[s], page, past[s] + t)
            for pl, x, ty in ((kp, k, Q8_0), (vp, v, F16)):
                for p, y in zip(pl, P.planes(x[s, t:t + 1], ty)):
                    p[r] = y[0]
    assert same(planes_of(kc), kp) and same(planes_of(vc), vp) and int(err) == 1


def test_append_broken_trees(mx):
    """A node whose way up meets no node before its own counts as padding: its row and query stay."""
    import torch
    T, page, HK, D = 9, 32, 2, 64
    rng = np.random.default_rng(2)
    parents = np.array([[-1, 0, 1, 3, 3, 8, -2, 1, 6], [-1, -1, 0, 0, 70, 4, 2 ** 31 - 1, -2 ** 31, 3]], np.int32)
    past, new = [3, 50], [9, 9]
    table, pages = tables(rng, past, new, page)
    kc, kp = cache_of(mx, Q4_0, pages * page, HK, D, rng)
    vc, vp = cache_of(mx, Q8_0, pages * page, HK, D, rng)
    k, v = (rng.standard_normal((2, T, HK, D)).astype(np.float32) for _ in range(2))
    freq = (10000.0 ** (-np.arange(32) / 32)).astype(np.float32)
    step = mx.KvStep(i32(table), i32(past), T, page, parents=i32(parents))
    err, q_out = zeros_i32(), torch.full((2, T, HK, D), 7.0, device="cuda")
    mx.kv_append(step, kc, vc, gpu(k), gpu(v), rope=mx.Rope(gpu(freq), neox=True), q=gpu(k), q_out=q_out, err=err)
    want = np.full((2, T, HK, D), 7.0, np.float32)
    for s in range(2):
        for t, way in enumerate(P.ways(parents[s], T)):
            if way is None:
                continue
            turned = P.rotate(k[s, t:t + 1], [past[s] + len(way) - 1], freq, True)
            want[s, t] = turned[0]
            r = P.row(table[s], page, past[s] + t)
            for pl, x, ty in ((kp, turned, Q4_0), (vp, v[s, t:t + 1], Q8_0)):
                for p, y in zip(pl, P.planes(x, ty)):
                    p[r] = y[0]
    assert same(planes_of(kc), kp) and same(planes_of(vc), vp) and np.array_equal(cpu(q_out), want) and int(err) == 1


# ---- attention ------------------------------------------------------------------------------

ATTEND = [  # S, T, tree, past, page, H, HK, D, DV
    (1, 1, False, [0], 32, 4, 2, 64, 64),
    (1, 1, False, [30], 32, 8, 2, 128, 128),
    (1, 1, False, [31], 32, 8, 8, 128, 128),
    (1, 1, False, [32], 64, 8, 1, 128, 128),
    (1, 1, False, [5000], 128, 8, 2, 128, 128),
    (4, 1, False, [0, 1, 63, 700], 64, 6, 2, 96, 96),
    (1, 16, True, [1500], 32, 4, 2, 256, 256),
    (3, 64, True, [0, 33, 900], 96, 8, 2, 64, 64),
    (2, 7, True, [0, 31], 32, 20, 1, 192, 128),
    (5, 13, True, [3, 0, 90, 200, 31], 32, 4, 4, 128, 96),
    (1, 130, False, [777], 64, 4, 2, 64, 32),
    (2, 40, False, [0, 2000], 256, 4, 1, 160, 128),
    (1, 33, False, [1], 32, 16, 2, 128, 64),
]


def attend_case(mx, kt, vt, case, seed=0, junk=0.05, new=None):
    S, T, is_tree, past, page, H, HK, D, DV = case
    rng = np.random.default_rng(seed + S * 1000 + T + D)
    if new is None:
        new = [T] if S == 1 else [T] + [int(n) for n in rng.integers(0, T + 1, S - 1)]
    table, pages = tables(rng, past, new, page)
    rows = pages * page
    seen = np.zeros(rows, bool)
    for s in range(S):
        seen[[P.row(table[s], page, j) for j in range(past[s] + new[s])]] = True
    caches = []
    for t, d in ((kt, D), (vt, DV)):
        c, pl = cache_of(mx, t, rows, HK, d, rng)
        pl[-1][~seen] = 0x7E00                       # what no sequence holds may be anything
        (c.q if t == F16 else c.d).copy_(gpu(pl[-1].view(np.float16)))
        caches.append((c, pl))
    q = rng.standard_normal((S, T, H, D)).astype(np.float32)
    parents = tree(rng, S, T) if is_tree else None
    step = mx.KvStep(i32(table), i32(past), T, page, n_new=i32(new), parents=None if parents is None else i32(parents))
    return dict(S=S, T=T, past=past, new=new, page=page, table=table, pages=pages, caches=caches, q=q, parents=parents, step=step, D=D, DV=DV, H=H,
                kt=kt, vt=vt)


def check_attend(c, got, scale, softcap=0.0, half=False):
    for s in range(c["S"]):
        want, tol = P.attend(c["q"][s].transpose(1, 0, 2).astype(np.float64), c["caches"][0][1], c["caches"][1][1], c["kt"], c["vt"], c["table"][s], c["page"],
                             c["pages"], c["past"][s], c["new"][s], None if c["parents"] is None else c["parents"][s], scale, softcap, c.get("cap"))
        if half:
            tol = tol + np.abs(want) * R.HALF + 2.0 ** -25
        d = np.abs(got[s] - want)
        over = float((d - tol).max(initial=-1.0)) if np.isfinite(d).all() else float("inf")
        assert over <= 1e-30, (s, over)


@pytest.mark.parametrize("kt,vt", ATTENDED, ids=lambda t: NAME[t])
@pytest.mark.parametrize("case", ATTEND, ids=lambda c: "S%dT%d%sD%d-%d" % (c[0], c[1], "t" if c[2] else "c", c[7], c[8]))
def test_attend(mx, form, kt, vt, case):
    import torch
    c = attend_case(mx, kt, vt, case)
    scale = float(np.float32(c["D"] ** -0.5))
    out = torch.full((c["S"], c["T"], c["H"], c["DV"]), float("nan"), device="cuda")
    err = zeros_i32()
    mx.flash_attn_paged(gpu(c["q"]).permute(0, 2, 1, 3), *[x[0] for x in c["caches"]], c["step"], scale, out=out, err=err)
    check_attend(c, cpu(out), scale)
    assert int(err) == 0


@pytest.mark.parametrize("kt,vt", ATTENDED, ids=lambda t: NAME[t])
@pytest.mark.parametrize("nsplit,max_kv", [(1, 0), (2, 0), (7, 0), (64, 0), (0, 2500), (0, 2405)])
def test_attend_splits_softcap_f16(mx, kt, vt, nsplit, max_kv):
    """Every split, plans for less than there is, fp16 queries and results, a soft-cap; the same bits twice."""
    import torch
    c = attend_case(mx, kt, vt, (3, 5, True, [2400, 0, 333], 32, 8, 2, 128, 128), seed=3)
    c["q"] = (3 * c["q"]).astype(np.float16)
    scale = float(np.float32(c["D"] ** -0.5))
    outs = []
    for _ in range(2):
        out = torch.full((3, 5, 8, 128), float("nan"), device="cuda", dtype=torch.float16)
        mx.flash_attn_paged(gpu(c["q"]).permute(0, 2, 1, 3), *[x[0] for x in c["caches"]], c["step"], scale, softcap=5.0, nsplit=nsplit, out=out, max_kv=max_kv)
        outs.append(cpu(out))
    assert np.array_equal(outs[0].view(np.uint16), outs[1].view(np.uint16))
    check_attend(c, outs[0].astype(np.float64), scale, 5.0, half=True)


ATTEND_FAULTS = {  # past, new, change of the table
    "past_negative": ([-1, 60], [3, 3], None),
    "past_behind": ([97, 60], [3, 3], None),
    "past_huge": ([2 ** 31 - 1, 60], [3, 3], None),
    "new_negative": ([50, 60], [-1, 3], None),
    "new_above": ([50, 60], [5, 3], None),
    "table_ends": ([95, 60], [3, 3], None),
    "page_negative": ([70, 60], [3, 3], (0, 1, -1)),
    "page_above": ([70, 60], [3, 3], (0, 2, 7)),
    "page_huge": ([70, 60], [3, 3], (0, 0, 2 ** 31 - 1)),
    "no_page": ([10, 60], [3, 3], (0, 0, 99)),
}


@pytest.mark.parametrize("mix", [(Q8_0, Q8_0), (Q4_0, Q4_0), (F16, F16)], ids=ids)
@pytest.mark.parametrize("name", ATTEND_FAULTS)
def test_attend_numbers_out_of_range(mx, form, mix, name):
    """Keys without a row count for nothing, and the flag is set."""
    past, new, change = ATTEND_FAULTS[name]
    T, page, H, HK, D = 3, 32, 4, 2, 64
    rng = np.random.default_rng(8)
    table = np.array([[0, 1, 2], [3, 4, 5]], np.int32)
    if change:
        table[change[0], change[1]] = change[2]
    caches = [cache_of(mx, t, 7 * page + 31, HK, D, rng) for t in mix]
    q = rng.standard_normal((2, T, H, D)).astype(np.float32)
    c = dict(S=2, T=T, past=past, new=new, page=page, table=table, pages=7, caches=caches, q=q, parents=None, kt=mix[0], vt=mix[1])
    err = zeros_i32()
    step = mx.KvStep(i32(table), i32(past), T, page, n_new=i32(new))
    got = mx.flash_attn_paged(gpu(q).permute(0, 2, 1, 3), caches[0][0], caches[1][0], step, 0.125, err=err)
    check_attend(c, cpu(got), 0.125)
    assert int(err) == 1


@pytest.mark.parametrize("mix", [(Q8_0, Q4_0), (F16, F16)], ids=ids)
@pytest.mark.parametrize("max_kv", [63, 64, 1, 40])
def test_attend_fewer_keys_than_held(mx, form, mix, max_kv):
    """Rows behind max_kv are not read, and the flag is set: a sequence that held more is as one without tokens."""
    T, page, H, HK, D = 3, 64, 4, 2, 64
    rng = np.random.default_rng(max_kv)
    past, new = [62, 10, 0], [3, 3, 2]
    table, pages = tables(rng, past, new, page)
    caches = [cache_of(mx, t, pages * page, HK, D, rng) for t in mix]
    q = rng.standard_normal((3, T, H, D)).astype(np.float32)
    err = zeros_i32()
    step = mx.KvStep(i32(table), i32(past), T, page, n_new=i32(new))
    got = cpu(mx.flash_attn_paged(gpu(q).permute(0, 2, 1, 3), caches[0][0], caches[1][0], step, 0.125, max_kv=max_kv, err=err))
    c = dict(S=3, T=T, past=past, new=new, page=page, table=table, pages=pages, caches=caches, q=q, parents=None, kt=mix[0], vt=mix[1], cap=max_kv)
    check_attend(c, got, 0.125)
    assert int(err) == 1


@pytest.mark.parametrize("mix", [(Q8_0, Q8_0), (Q4_0, Q4_0), (F16, F16)], ids=ids)
def test_attend_broken_trees_and_wild_queries(mx, mix):
    """Nodes without a way up are zeros; infinities and NaN in one token's query stay in its rows."""
    import torch
    T, page, H, HK, D = 9, 32, 4, 2, 64
    rng = np.random.default_rng(2)
    parents = np.array([[-1, 0, 1, 3, 3, 8, -2, 1, 6], [-1, -1, 0, 0, 70, 4, 2 ** 31 - 1, -2 ** 31, 3]], np.int32)
    past, new = [3, 50], [9, 9]
    table, pages = tables(rng, past, new, page)
    caches = [cache_of(mx, t, pages * page, HK, D, rng) for t in mix]
    q = rng.standard_normal((2, T, H, D)).astype(np.float32)
    c = dict(S=2, T=T, past=past, new=new, page=page, table=table, pages=pages, caches=caches, q=q, parents=parents, kt=mix[0], vt=mix[1])
    err = zeros_i32()
    step = mx.KvStep(i32(table), i32(past), T, page, parents=i32(parents))
    got = cpu(mx.flash_attn_paged(gpu(q).permute(0, 2, 1, 3), caches[0][0], caches[1][0], step, 0.125, err=err))
    check_attend(c, got, 0.125)
    assert int(err) == 1
    assert not got[0, [3, 4, 5, 6, 8]].any() and not got[1, [4, 5, 6, 7]].any()
    wild = q.copy()
    wild[0, 0, 1, 5], wild[1, 1] = np.nan, np.inf
    wild[0, 6] = np.nan                              # padding's query
    again = cpu(mx.flash_attn_paged(gpu(wild).permute(0, 2, 1, 3), caches[0][0], caches[1][0], step, 0.125))
    keep = np.ones(q.shape[:3], bool)
    keep[0, 0, 1] = keep[1, 1] = False
    assert np.array_equal(again[keep], got[keep]) and np.isnan(again[0, 0, 1]).all()


@pytest.mark.parametrize("mix", [(Q8_0, Q8_0), (Q4_0, Q4_0), (F16, F16)], ids=ids)
def test_attend_keys_with_nan_scales(mx, mix):
    """A drafted key with a scale that is no number makes exactly the rows of the tokens that see it NaN."""
    T, page, H, HK, D = 12, 32, 2, 1, 128
    rng = np.random.default_rng(6)
    parents = tree(rng, 1, T)
    past = [70]
    table, pages = tables(rng, past, [T], page)
    for which in range(2):
        caches = [cache_of(mx, t, pages * page, HK, D, rng) for t in mix]
        c, at = caches[which][0], P.row(table[0], page, past[0] + 2)
        if c.type == F16:
            c.q[at, 0, 40] = float("nan")
        else:
            c.d[at, 0, 1] = float("inf")
        q = rng.standard_normal((1, T, H, D)).astype(np.float32)
        step = mx.KvStep(i32(table), i32(past), T, page, parents=i32(parents))
        got = cpu(mx.flash_attn_paged(gpu(q).permute(0, 2, 1, 3), caches[0][0], caches[1][0], step, 0.09))
        sees = np.array([2 in w for w in P.ways(parents[0], T)])
        assert sees.any() and not sees.all()
        assert np.isnan(got[0, sees]).all() and np.isfinite(got[0, ~sees]).all()


@pytest.mark.parametrize("vt", [Q8_0, Q4_0], ids=ids)
@pytest.mark.parametrize("DV", [64, 128, 256])
@pytest.mark.parametrize("T", [1, 9])
@pytest.mark.parametrize("ratio", [1e2, 1e4, 1e6])
def test_attend_blocks_of_a_key_apart(mx, form, vt, DV, T, ratio):
    """V's blocks of dims whose values are `ratio` apart: each is as good as its own values allow."""
    H, HK, KV, page, D = 8, 2, 400, 32, 64 if DV < 256 else 256
    rng = np.random.default_rng(DV + T)
    table, pages = tables(rng, [KV - T], [T], page)
    at = np.array([P.row(table[0], page, j) for j in range(KV)])
    kc, kp = cache_of(mx, Q8_0, pages * page, HK, D, rng)
    x = rng.standard_normal((pages * page, HK, DV // 32, 32))
    x *= 8000.0 / np.abs(x).max(-1)[..., None]
    x[:, :, 1::2] /= ratio
    vq, vd = R.quantize(x.reshape(-1, HK, DV), vt)
    q = rng.standard_normal((1, T, H, D)).astype(np.float32)
    mask = np.where(np.arange(KV) <= KV - T + np.arange(T)[:, None], 0.0, -np.inf)
    kn, vn = P.cache_values([p[at] for p in kp], Q8_0), R.values(vq, vd, vt)[at]
    want, limit = kv_norm.attention(q[0].transpose(1, 0, 2), kn.transpose(1, 0, 2), vn.transpose(1, 0, 2), mask, D ** -0.5, vd=vd[at].transpose(1, 0, 2))
    step = mx.KvStep(i32(table), i32([KV - T]), T, page)
    for ns in (0, 1, 3):
        got = cpu(mx.flash_attn_paged(gpu(q).permute(0, 2, 1, 3), kc, mx.KvCache(vt, gpu(vq), gpu(vd)), step, D ** -0.5, nsplit=ns))[0]
        assert kv_norm.ratio(got, want, limit) <= 1, (ns, kv_norm.ratio(got, want, limit))


@pytest.mark.parametrize("kt,vt", [(Q8_0, Q4_0), (F16, F16)], ids=lambda t: NAME[t])
def test_attend_far_rows(mx, kt, vt):
    """Pages past 2^31 bytes and values of the cache."""
    import torch
    H, HK, D, page = 8, 8, 128, 64
    rows = (1 << 21) + 64 * 40                       # times 1024 codes
    kc, vc = mx.kv_cache(kt, rows, HK, D), mx.kv_cache(vt, rows, HK, D)
    rng = np.random.default_rng(1)
    pages = np.array([[rows // page - 1, 1, rows // page - 20, (1 << 21) // page]], np.int32)
    n = 4 * page - 3
    at = np.array([P.row(pages[0], page, j) for j in range(n)])
    k, v = (rng.standard_normal((1, n, HK, D)).astype(np.float32) for _ in range(2))
    first = mx.KvStep(i32(pages), i32([0]), n, page)
    mx.kv_append(first, kc, vc, gpu(k), gpu(v))
    got = mx.get_rows([kc, vc], gpu(at))
    kp, vp = P.planes(k[0], kt), P.planes(v[0], vt)
    assert np.array_equal(cpu(got[0]), P.cache_values(kp, kt).astype(np.float32))
    assert np.array_equal(cpu(got[1]), P.cache_values(vp, vt).astype(np.float32))
    q = rng.standard_normal((1, 1, H, D)).astype(np.float32)
    step = mx.KvStep(i32(pages), i32([n - 1]), 1, page)
    out = cpu(mx.flash_attn_paged(gpu(q).permute(0, 2, 1, 3), kc, vc, step, 0.09))
    want, tol = R.attention(q[0].transpose(1, 0, 2).astype(np.float64), P.cache_values(kp, kt).transpose(1, 0, 2), P.cache_values(vp, vt).transpose(1, 0, 2), None, 0.09)
    assert (np.abs(out[0] - want) <= tol).all()


# ---- keep -----------------------------------------------------------------------------------

@pytest.mark.parametrize("t", [Q8_0, Q4_0, F16], ids=ids)
@pytest.mark.parametrize("S,T,A,H,D,page", [(1, 2, 1, 1, 32, 32), (1, 64, 64, 8, 128, 32), (7, 33, 9, 3, 96, 64), (3, 200, 17, 64, 128, 96)])
def test_keep_bits(mx, t, S, T, A, H, D, page):
    """Kept rows in order, bit by bit; everything else as it was. Paths that step on rows they write, and whole ones."""
    rng = np.random.default_rng(T + A)
    past = [int(n) for n in rng.integers(0, 300, S)]
    new = [T] + [int(n) for n in rng.integers(0, T + 1, S - 1)]
    keep = [min(n, A) if i % 3 == 0 else int(rng.integers(0, min(n, A) + 1)) for i, n in enumerate(new)]
    path = np.full((S, A), -5, np.int32)
    for s in range(S):
        path[s, :keep[s]] = np.sort(rng.permutation(new[s])[:keep[s]])
    table, pages = tables(rng, past, new, page)
    (c1, p1), (c2, p2) = cache_of(mx, t, pages * page, H, D, rng), cache_of(mx, Q8_0, pages * page + 3, 2, 64, rng)
    step = mx.KvStep(i32(table), i32(past), T, page, n_new=i32(new))
    err = zeros_i32()
    mx.kv_keep(step, [c1, c2], i32(path), n_keep=i32(keep), err=err)
    for s in range(S):
        for i in range(keep[s]):
            src, dst = P.row(table[s], page, past[s] + path[s, i]), P.row(table[s], page, past[s] + i)
            for p in p1 + p2:
                p[dst] = p[src]
    assert same(planes_of(c1), p1) and same(planes_of(c2), p2) and int(err) == 0


KEEP_FAULTS = {  # past, new, keep, path of sequence 0, change of the table
    "falling": (5, 8, 3, [1, 4, 3], None), "twice": (5, 8, 3, [1, 1, 2], None), "before": (5, 8, 2, [-1, 2], None),
    "padding": (5, 8, 3, [1, 2, 8], None), "many": (5, 8, 4, [1, 2, 3], None), "negative": (5, 8, -1, [1, 2, 3], None),
    "past": (-1, 8, 3, [1, 2, 3], None), "new": (5, 11, 3, [1, 2, 3], None), "behind": (90, 8, 3, [1, 2, 7], None),
    "no_source": (28, 8, 3, [0, 1, 7], (0, 1, 9)), "no_row": (28, 8, 3, [5, 6, 7], (0, 0, -1)),
}


@pytest.mark.parametrize("name", KEEP_FAULTS)
def test_keep_numbers_out_of_range(mx, name):
    """The sequence stays as it is, the other one's rows move, and the flag is set."""
    past, new, keep, path, change = KEEP_FAULTS[name]
    rng = np.random.default_rng(3)
    table = np.array([[0, 1, 2], [3, 4, 5]], np.int32)
    if change:
        table[change[0], change[1]] = change[2]
    c, p = cache_of(mx, Q4_0, 7 * 32 + 8, 2, 64, rng)
    step = mx.KvStep(i32(table), i32([past, 20]), 10, 32, n_new=i32([new, 10]))
    err = zeros_i32()
    mx.kv_keep(step, [c], i32([path + [0] * (3 - len(path)), [2, 5, 9]]), n_keep=i32([keep, 3]), err=err)
    for i, u in enumerate([2, 5, 9]):
        for x in p:
            x[P.row(table[1], 32, 20 + i)] = x[P.row(table[1], 32, 20 + u)]
    assert same(planes_of(c), p) and int(err) == 1


# ---- the three of them ------------------------------------------------------------------------

class Loop:
    """A drafting loop over two sequences, as a program runs it: append, attend, keep; lengths on the device."""

    def __init__(self, mx, kt, vt, seed):
        import torch
        self.mx, self.S, self.T, self.H, self.HK, self.D, self.page = mx, 2, 6, 4, 2, 64, 32
        self.kt, self.vt = kt, vt
        rng = self.rng = np.random.default_rng(seed)
        self.table = np.array([rng.permutation(8)[:4], [8, 12, 9, 10]], np.int32)
        self.past = np.array([29, 0], np.int32)
        self.kc, self.kp = cache_of(mx, kt, 13 * 32, self.HK, self.D, rng)
        self.vc, self.vp = cache_of(mx, vt, 13 * 32, self.HK, self.D, rng)
        self.freq = (10000.0 ** (-np.arange(16) / 16)).astype(np.float32)
        shape = (self.S, self.T)
        self.dev = dict(table=i32(self.table), past=i32(self.past), new=i32([6, 6]), parents=i32(np.zeros(shape)), path=i32(np.zeros((2, 4))), keep=i32([0, 0]),
                        q=torch.zeros(*shape, self.H, self.D, device="cuda"), k=torch.zeros(*shape, self.HK, self.D, device="cuda"),
                        v=torch.zeros(*shape, self.HK, self.D, device="cuda"), qr=torch.zeros(*shape, self.H, self.D, device="cuda", dtype=torch.float16),
                        out=torch.zeros(*shape, self.H, self.D, device="cuda"), err=zeros_i32())
        d = self.dev
        self.step = mx.KvStep(d["table"], d["past"], self.T, self.page, n_new=d["new"], parents=d["parents"])
        self.rope = mx.Rope(gpu(self.freq), neox=True)
        need = mx.flash_attn_paged_workspace(d["qr"].permute(0, 2, 1, 3), self.kc, self.vc, self.step, d["out"])
        self.ws = torch.empty(need, dtype=torch.uint8, device="cuda")

    def calls(self):
        d = self.dev
        self.mx.kv_append(self.step, self.kc, self.vc, d["k"], d["v"], rope=self.rope, q=d["q"], q_out=d["qr"], err=d["err"])
        self.mx.flash_attn_paged(d["qr"].permute(0, 2, 1, 3), self.kc, self.vc, self.step, 0.125, out=d["out"], workspace=self.ws, err=d["err"])
        self.mx.kv_keep(self.step, [self.kc, self.vc], d["path"], n_keep=d["keep"], err=d["err"])
        d["past"].add_(d["keep"])

    def inputs(self):
        rng, d = self.rng, self.dev
        new = rng.integers(1, self.T + 1, self.S).astype(np.int32)
        parents = tree(rng, self.S, self.T)
        keep, path = np.zeros(2, np.int32), np.zeros((2, 4), np.int32)
        for s in range(2):
            way = P.ways(parents[s], new[s])[int(rng.integers(0, new[s]))][::-1][:4]
            keep[s], path[s, :len(way)] = len(way), way
        self.now = dict(new=new, parents=parents, keep=keep, path=path)
        for n, x in self.now.items():
            d[n].copy_(gpu(x))
        for n in ("q", "k", "v"):
            self.now[n] = rng.standard_normal(tuple(d[n].shape)).astype(np.float32)
            d[n].copy_(gpu(self.now[n]))

    def check(self):
        x, d = self.now, self.dev
        out = cpu(d["out"])
        for s in range(self.S):
            n, past, tab = int(x["new"][s]), int(self.past[s]), self.table[s]
            at = [P.row(tab, self.page, past + t) for t in range(n)]
            pos = [past + len(w) - 1 for w in P.ways(x["parents"][s], n)]
            for p, y in zip(self.kp, P.planes(P.rotate(x["k"][s, :n], pos, self.freq, True), self.kt)):
                p[at] = y
            for p, y in zip(self.vp, P.planes(x["v"][s, :n], self.vt)):
                p[at] = y
            q = np.zeros((self.T, self.H, self.D))
            q[:n] = P.rotate(x["q"][s, :n], pos, self.freq, True).astype(np.float16)
            want, tol = P.attend(q.transpose(1, 0, 2), self.kp, self.vp, self.kt, self.vt, tab, self.page, 13, past, n, x["parents"][s], 0.125)
            assert (np.abs(out[s] - want) <= tol + 1e-30).all()
            for i in range(int(x["keep"][s])):
                for p in self.kp + self.vp:
                    p[P.row(tab, self.page, past + i)] = p[P.row(tab, self.page, past + int(x["path"][s, i]))]
            self.past[s] += x["keep"][s]
        assert same(planes_of(self.kc), self.kp) and same(planes_of(self.vc), self.vp)
        assert np.array_equal(cpu(d["past"]), self.past) and int(d["err"]) == 0


@pytest.mark.parametrize("mix", [(Q8_0, Q8_0), (Q4_0, Q8_0), (F16, F16)], ids=ids)
def test_loop(mx, mix):
    loop = Loop(mx, *mix, seed=5)
    for _ in range(8):
        loop.inputs()
        loop.calls()
        loop.check()


@pytest.mark.parametrize("mix", [(Q8_0, Q8_0), (Q4_0, Q8_0), (F16, F16)], ids=ids)
def test_loop_captured(mx, mix):
    """The step captured once follows the lengths, trees and tables of every replay; eager steps in between."""
    import torch
    loop = Loop(mx, *mix, seed=6)
    loop.inputs()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        loop.calls()
    stream.synchronize()
    loop.check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        loop.calls()
    for i in range(8):
        loop.inputs()
        torch.cuda.synchronize()
        if i % 3 == 2:
            loop.calls()
        else:
            graph.replay()
        loop.check()


@pytest.mark.parametrize("mix", [(Q8_0, Q4_0), (F16, F16)], ids=ids)
def test_lengths_that_change_inside_a_graph(mx, mix):
    """Several steps in one graph: each call sees the lengths that the call before it left."""
    import torch
    H, HK, D, page, n = 4, 2, 64, 32, 5
    rng = np.random.default_rng(9)
    table, pages = tables(rng, [90], [20 * n], page)
    caches = [cache_of(mx, t, pages * page, HK, D, rng) for t in mix]
    q, k, v = (rng.standard_normal((n, 1, 1, h, D)).astype(np.float32) for h in (H, HK, HK))
    dq, dk, dv = gpu(q), gpu(k), gpu(v)
    past = i32([60])
    step = mx.KvStep(i32(table), past, 1, page)
    kc, vc = caches[0][0], caches[1][0]
    outs = [torch.zeros(1, 1, H, D, device="cuda") for _ in range(n)]
    ws = torch.empty(mx.flash_attn_paged_workspace(dq[0].permute(0, 2, 1, 3), kc, vc, step, outs[0]), dtype=torch.uint8, device="cuda")

    def calls():
        for i in range(n):
            mx.kv_append(step, kc, vc, dk[i], dv[i])
            mx.flash_attn_paged(dq[i].permute(0, 2, 1, 3), kc, vc, step, 0.125, out=outs[i], workspace=ws)
            past.add_(1)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        calls()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        calls()
    at = 60 + n                                     # the eager steps; capturing runs nothing
    for _ in range(4):
        for pl, x, t in ((caches[0][1], k, mix[0]), (caches[1][1], v, mix[1])):
            pl[:] = planes_of(kc if pl is caches[0][1] else vc)
        graph.replay()
        got = [cpu(o) for o in outs]
        for i in range(n):
            r = P.row(table[0], page, at + i)
            for pl, x, t in ((caches[0][1], k, mix[0]), (caches[1][1], v, mix[1])):
                for p, y in zip(pl, P.planes(x[i, 0], t)):
                    p[r] = y[0]
            want, tol = P.attend(q[i, 0].transpose(1, 0, 2).astype(np.float64), caches[0][1], caches[1][1], *mix, table[0], page, pages, at + i, 1, None, 0.125)
            assert (np.abs(got[i][0] - want) <= tol).all()
        at += n
        assert int(past[0]) == at


def test_two_streams_at_once(mx):
    """Calls in flight on two streams, a workspace each, over one cache."""
    import torch
    c = attend_case(mx, Q8_0, Q8_0, (4, 6, True, [3000, 2500, 100, 0], 32, 8, 2, 128, 128), seed=2)
    q = gpu(c["q"]).permute(0, 2, 1, 3)
    caches = [x[0] for x in c["caches"]]
    want = cpu(mx.flash_attn_paged(q, *caches, c["step"], 0.09))
    outs = [torch.zeros(4, 6, 8, 128, device="cuda") for _ in range(2)]
    need = mx.flash_attn_paged_workspace(q, *caches, c["step"], outs[0])
    ws = [torch.empty(need, dtype=torch.uint8, device="cuda") for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                mx.flash_attn_paged(q, *caches, c["step"], 0.09, out=outs[i], workspace=ws[i])
    assert all(np.array_equal(cpu(o), want) for o in outs)

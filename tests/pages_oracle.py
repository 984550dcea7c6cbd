"""A KV cache in pages in plain numpy: rows of positions, trees of new tokens, the position rotation with the roundings that the
definition names, and attention over the rows that a token sees, in 64 bits (kv_oracle holds the formats and the bound of
fp16 operands)."""
import numpy as np

import kv_oracle as R

F16 = 1


def row(table, page, j):
    return int(table[j // page]) * page + j % page


def ways(parents, n):
    """For each of n tokens the tokens on its way up, itself first; None where the way meets a number that is no
    token before."""
    found = []
    for t in range(n):
        up = t - 1 if parents is None else int(parents[t])
        if up == -1:
            found.append([t])
        else:
            found.append([t] + found[up] if 0 <= up < t and found[up] is not None else None)
    return found


def f32(a):
    return np.asarray(a, dtype=np.float64).astype(np.float32).astype(np.float64)


def rotate(x, pos, freq, neox, mscale=1.0):
    """x [n][H][D] at positions pos [n], freq f32 [n_rot / 2]: every product and sum rounded to f32."""
    x = x.astype(np.float32).astype(np.float64)
    y = x.copy()
    half = len(freq)
    a = np.arange(half) if neox else 2 * np.arange(half)
    b = a + (half if neox else 1)
    th = np.asarray(pos, np.float64)[:, None, None] * freq.astype(np.float64)
    c, s = f32(np.cos(th) * np.float64(np.float32(mscale))), f32(np.sin(th) * np.float64(np.float32(mscale)))
    y[..., a] = f32(f32(x[..., a] * c) - f32(x[..., b] * s))
    y[..., b] = f32(f32(x[..., a] * s) + f32(x[..., b] * c))
    return y.astype(np.float32)


def planes(x, t):
    """The planes of stored rows, as raw integers."""
    if t == F16:
        with np.errstate(over="ignore"):
            return [x.astype(np.float16).view(np.uint16)]
    q, d = R.quantize(x, t)
    return [q, d.view(np.uint16)]


def cache_values(pl, t):
    if t == F16:
        return pl[0].view(np.float16).astype(np.float64)
    return R.held(pl[0], pl[1].view(np.float16), t)


def attend(q, kp, vp, kt, vt, table, page, n_pages, n_past, n_new, parents, scale, softcap=0.0, most=None):
    """q [H][T][D] of one sequence, planes of the caches -> (dst [T][H][DV], bound) as kv_oracle.attention; most: logical
    rows that count at most."""
    H, T, D = q.shape
    cap = min(len(table) * page, most or 1 << 40)
    fresh = max(0, min(T, n_new)) if 0 <= n_past <= cap else 0
    n = min(cap, n_past + fresh) if fresh else 0
    DV = vp[0].shape[-1] * (2 if vt == R.Q4_0 else 1)
    out, tol = np.zeros((T, H, DV)), np.zeros((T, H, DV))
    if not n:
        return out, tol
    have = np.array([0 <= table[j // page] < n_pages for j in range(n)])
    rows = np.array([row(table, page, j) if ok else 0 for j, ok in enumerate(have)])
    k = cache_values([p[rows] for p in kp], kt).transpose(1, 0, 2)
    v = cache_values([p[rows] for p in vp], vt).transpose(1, 0, 2)
    mask = np.full((T, n), -np.inf)
    for t, way in enumerate(ways(parents, fresh)):
        if way is None:
            continue
        mask[t, :n_past] = 0
        at = [n_past + u for u in way if n_past + u < n]
        mask[t, at] = 0
        mask[t, ~have] = -np.inf
    return R.attention(q, k, v, mask, scale, softcap)

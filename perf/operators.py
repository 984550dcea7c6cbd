"""The operators on a KV cache held in 8 or 4 bits, as cases that can be timed and checked.

Three operators of ggml_mi355x, as a decoder layer uses them one after the other:
  store   SET_ROWS: a layer's new keys and values, quantized into the rows of its cache that an
          index names (one call for both), then read back
  load    GET_ROWS: rows of the cache as plain values
  attn    FLASH_ATTN_EXT over the quantized cache, from a single token to a prefill's micro-batch
A cache is two planes with the same element strides: the codes (Q8_0: an int8 a value; Q4_0: 16
bytes a block of 32, value j in the low nibble of byte j, value j + 16 in the high one) and the
blocks' fp16 scales. Q8_0 stands for d * code, Q4_0 for d * (code - 8).
Head counts and dims are those of the 8B prefill, the attention tests (64, 96, 192 / 128, 256) and
the benchmark; activations are N(0, 1), as after a norm.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

Q4_0, Q8_0 = "Q4_0", "Q8_0"
DEV = "cuda"


# ---- cases ---------------------------------------------------------------------------------

def listed():
    return [
        # one generated token's K and V of an 8B layer: latency counts
        dict(name="store_token_q8_0", op="store", n=1, rows=4096, HK=8, dk=128, dv=128, kt=Q8_0, vt=Q8_0, src="F32"),
        # a 512-token micro-batch of the same layer in 4 bits
        dict(name="store_batch_q4_0", op="store", n=512, rows=8192, HK=8, dk=128, dv=128, kt=Q4_0, vt=Q4_0, src="F32"),
        # a long ragged prompt from fp16 projections, keys in 8 bits and values in 4
        dict(name="store_ragged_k8v4", op="store", n=4091, rows=16384, HK=8, dk=128, dv=128, kt=Q8_0, vt=Q4_0, src="F16"),
        # some scattered positions, for re-rotating them
        dict(name="load_rows_q4_0", op="load", n=333, rows=4096, HK=8, dk=64, dv=64, kt=Q4_0, vt=Q4_0, dst="F32"),
        # a whole context as fp16, as for a copy of the sequence
        dict(name="load_context_q8_0", op="load", n=32768, rows=32768, HK=8, dk=128, dv=128, kt=Q8_0, vt=Q8_0, dst="F16"),
        # one token early in a conversation
        dict(name="decode_q8_0_kv1000", op="attn", S=1, T=1, KV=1000, H=32, HK=8, dk=128, dv=128, kt=Q8_0, vt=Q8_0, q="F32", softcap=0.0),
        # one token deep in a long context
        dict(name="decode_q4_0_kv32768", op="attn", S=1, T=1, KV=32768, H=32, HK=8, dk=128, dv=128, kt=Q4_0, vt=Q4_0, q="F32", softcap=0.0),
        # 32 sequences of different lengths served together
        dict(name="decode_32seq_q8_0", op="attn", S=32, T=1, KV=4096, H=32, HK=8, dk=128, dv=128, kt=Q8_0, vt=Q8_0, q="F16", softcap=0.0),
        # five drafted tokens to verify, heads of 256 with a soft-cap
        dict(name="draft5_k8v4_d256", op="attn", S=1, T=5, KV=16384, H=16, HK=8, dk=256, dv=256, kt=Q8_0, vt=Q4_0, q="F32", softcap=50.0),
        # a short ragged prompt of a small model
        dict(name="prompt100_q4_0_d64", op="attn", S=1, T=100, KV=1531, H=32, HK=8, dk=64, dv=64, kt=Q4_0, vt=Q4_0, q="F32", softcap=0.0),
        # the 8B model at the last micro-batch of a 2048-token prefill
        dict(name="prefill_q8_0_kv2048", op="attn", S=1, T=512, KV=2048, H=32, HK=8, dk=128, dv=128, kt=Q8_0, vt=Q8_0, q="F32", softcap=0.0),
        # the same model deep in a long context, in 4 bits
        dict(name="prefill_q4_0_kv8192", op="attn", S=1, T=512, KV=8192, H=32, HK=8, dk=128, dv=128, kt=Q4_0, vt=Q4_0, q="F32", softcap=0.0),
    ]


def _log(rng, lo, hi):
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["store", "load", "attn", "attn", "attn", "attn"])
    kt, vt = rng.choice([(Q8_0, Q8_0), (Q4_0, Q4_0), (Q8_0, Q4_0), (Q4_0, Q8_0)])
    if op == "attn":
        dk, dv, H, HK = rng.choice([(64, 64, 32, 8), (96, 96, 32, 32), (128, 128, 32, 8), (128, 128, 32, 4), (128, 128, 16, 16),
                                    (192, 128, 16, 16), (256, 256, 16, 8)])
        S = rng.choice([1, 1, 1, _log(rng, 2, 32)])
        T = rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 64, 512)]) if S == 1 else rng.choice([1, 1, _log(rng, 2, 16)])
        most = min(32 * 4096 * 8 * 256 // (S * HK * (dk + dv)), 512 * 8192 * 32 * 256 // (S * T * H * (dk + dv)), 32768)
        return dict(op=op, S=S, T=T, KV=_log(rng, 17, most), H=H, HK=HK, dk=dk, dv=dv, kt=kt, vt=vt,
                    q=rng.choice(["F32", "F16"]), softcap=rng.choice([0.0, 0.0, 0.0, 50.0]))
    dk, dv, HK = rng.choice([(64, 64, 8), (96, 96, 32), (128, 128, 8), (128, 128, 16), (192, 128, 16), (256, 256, 8)])
    hi = 32768 * 8 * 256 // (HK * (dk + dv))
    if op == "store":
        n = _log(rng, 1, min(4096, hi))
        return dict(op=op, n=n, rows=n + _log(rng, 1, 8192), HK=HK, dk=dk, dv=dv, kt=kt, vt=vt, src=rng.choice(["F32", "F16"]))
    dst = rng.choice(["F32", "F16"])
    n = _log(rng, 1, hi if dst == "F16" else hi // 2)
    return dict(op=op, n=n, rows=n + rng.choice([0, _log(rng, 1, 4096)]), HK=HK, dk=dk, dv=dv, kt=kt, vt=vt, dst=dst)


def _lengths(case):
    """Cached positions of each sequence: all of them for one, spread over (0, KV] for several."""
    S, KV = case["S"], case["KV"]
    return [KV] if S == 1 else [max(1, round(KV * (1 - (0.618034 * s) % 1.0))) for s in range(S)]


def _bits(t):
    return {Q8_0: 8.5, Q4_0: 4.5, "F16": 16.0, "F32": 32.0}[t]


def work(case):
    HK, dk, dv = case["HK"], case["dk"], case["dv"]
    held = (dk * _bits(case["kt"]) + dv * _bits(case["vt"])) / 8      # bytes of one position of one KV head
    if case["op"] == "store":    # sources in, rows written, rows read, their values out
        return {"bytes": case["n"] * (HK * (2 * held + (dk + dv) * (_bits(case["src"]) / 8 + 4)) + 8),
                "flops": 3.0 * case["n"] * HK * (dk + dv)}
    if case["op"] == "load":
        return {"bytes": case["n"] * (HK * (held + (dk + dv) * _bits(case["dst"]) / 8) + 4), "flops": 1.0 * case["n"] * HK * (dk + dv)}
    S, T, H, KV = case["S"], case["T"], case["H"], case["KV"]
    pairs = sum(max(0, n - T + t + 1) for n in _lengths(case) for t in range(T))
    io = S * T * H * (dk * _bits(case["q"]) / 8 + dv * 2) + S * T * KV * 2
    return {"bytes": io + sum(_lengths(case)) * HK * held, "flops": 2.0 * pairs * H * (dk + dv)}


# ---- inputs --------------------------------------------------------------------------------

def _random_cache(g, t, *shape):
    """(codes, scales) of a cache holding N(0, 1) values, every block scaled to its largest."""
    x = torch.randn(*shape[:-1], shape[-1] // 32, 32, generator=g, device=DEV)
    d = (x.abs().amax(-1, keepdim=True) / (127.0 if t == Q8_0 else 8.0)).half()
    x = x.div_(d.float()).round_()
    if t == Q8_0:
        return x.clamp_(-127, 127).to(torch.int8).reshape(*shape), d.squeeze(-1)
    u = x.clamp_(-8, 7).add_(8).to(torch.uint8)
    return (u[..., :16] | (u[..., 16:] << 4)).reshape(*shape[:-1], shape[-1] // 2), d.squeeze(-1)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    s = dict(case=dict(case))
    HK, dk, dv = case["HK"], case["dk"], case["dv"]
    if case["op"] == "attn":
        S, T, KV, H = case["S"], case["T"], case["KV"], case["H"]
        s["k"] = _random_cache(g, case["kt"], S, KV, HK, dk)
        s["v"] = _random_cache(g, case["vt"], S, KV, HK, dv)
        q = torch.randn(S, T, H, dk, generator=g, device=DEV)
        s["q"] = (q.half() if case["q"] == "F16" else q).permute(0, 2, 1, 3)
        # causal, the last query of a sequence sees all of it; rows padded as ggml pads them
        n = torch.tensor(_lengths(case), device=DEV)[:, None, None]
        j = torch.arange((KV + 63) // 64 * 64, device=DEV)[None, None, :]
        t = torch.arange(T, device=DEV)[None, :, None]
        s["mask"] = torch.zeros(S, T, j.shape[-1], dtype=torch.float16, device=DEV).masked_fill_(j > n - T + t, float("-inf"))
        return s
    n, rows = case["n"], case["rows"]
    s["k"] = _random_cache(g, case["kt"], rows, HK, dk)
    s["v"] = _random_cache(g, case["vt"], rows, HK, dv)
    if case["op"] == "store":
        src = torch.float16 if case["src"] == "F16" else torch.float32
        s["xk"] = torch.randn(n, HK, dk, generator=g, device=DEV).to(src)
        s["xv"] = torch.randn(n, HK, dv, generator=g, device=DEV).to(src)
    at = torch.randperm(rows, generator=g, device=DEV)[:n]
    s["idx"] = at if case["op"] == "store" else (at.sort().values if n < rows else torch.arange(rows, device=DEV)).int()
    return s


# ---- one pass ------------------------------------------------------------------------------

def _plain_codes(x, t):
    """The codes and scales of x [..., D] by the formats' definition: a block's scale is max|x| / 127
    (Q8_0) or the value of largest magnitude (the first of equals) / -8 (Q4_0), codes are x times the
    reciprocal of the scale, rounded half away from zero. Each product and quotient is a 32-bit one;
    they are formed in 64 bits and rounded, since a value next to a border changes its code."""
    b = x.double().reshape(*x.shape[:-1], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    if t == Q8_0:
        d = (top / 127.0).float()
    else:
        first = (b.abs() == top).to(torch.uint8).argmax(-1, keepdim=True)
        d = (b.gather(-1, first) / -8.0).float()
    r = torch.where(d == 0, 0.0, 1.0 / d.double()).float()
    y = (b * r.double()).float()
    if t == Q8_0:
        c = (y.double() + torch.where(y < 0, -0.5, 0.5).double()).trunc().to(torch.int8).reshape(x.shape)
        return c, d.squeeze(-1).half()
    u = (y + 8.5).trunc().clamp(0, 15).to(torch.uint8)
    return (u[..., :16] | (u[..., 16:] << 4)).reshape(*x.shape[:-1], -1), d.squeeze(-1).half()


def _plain_values(codes, d, t):
    if t == Q8_0:
        c = codes.float().reshape(*d.shape, 32)
    else:
        u = codes.reshape(*d.shape, 16)
        c = torch.cat([u & 15, u >> 4], -1).float() - 8.0
    return (c * d.float()[..., None]).flatten(-2)


def _plain_attn(s):
    case = s["case"]
    S, T, KV, H, HK, dk, dv = (case[n] for n in ("S", "T", "KV", "H", "HK", "dk", "dv"))
    k = _plain_values(*s["k"], case["kt"]).transpose(1, 2).contiguous()            # [S][HK][KV][dk]
    v = _plain_values(*s["v"], case["vt"]).transpose(1, 2).contiguous()
    q = s["q"].float().reshape(S, HK, H // HK * T, dk)
    p = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(1.0 / math.sqrt(dk)).view(S, H, T, KV)
    if case["softcap"]:
        p = p.div_(case["softcap"]).tanh_().mul_(case["softcap"])
    p = p.add_(s["mask"][:, None, :, :KV])
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    den = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(S, HK, H // HK * T, KV), v).view(S, H, T, dv)
    o = torch.where(den > 0, o / den, 0.0)
    return o.transpose(1, 2).contiguous().half()


def _mx():
    at = os.path.join(os.getcwd(), "ggml-rocket_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import ggml_mi355x
    return ggml_mi355x


def _cache(mx, planes, t):
    return mx.KvCache(mx.Q8_0 if t == Q8_0 else mx.Q4_0, *planes)


def run(s):
    case = s["case"]
    if not own:
        if case["op"] == "attn":
            return _plain_attn(s)
        at = s["idx"].long()
        if case["op"] == "store":
            for planes, x, t in ((s["k"], s["xk"], case["kt"]), (s["v"], s["xv"], case["vt"])):
                codes, d = _plain_codes(x, t)
                planes[0][at] = codes
                planes[1][at] = d
        dst = torch.float16 if case.get("dst") == "F16" else torch.float32
        return [_plain_values(c[at], d[at], t).to(dst) for (c, d), t in ((s["k"], case["kt"]), (s["v"], case["vt"]))]
    mx = _mx()
    if "caches" not in s:      # a program keeps its caches, its workspace and its output buffers
        s["caches"] = _cache(mx, s["k"], case["kt"]), _cache(mx, s["v"], case["vt"])
        if case["op"] == "attn":
            S, T, H, dv = (case[n] for n in ("S", "T", "H", "dv"))
            s["kv"] = [c.permute(0, 2, 1, 3) for c in s["caches"]]
            s["out"] = torch.empty(S, T, H, dv, dtype=torch.float16, device=DEV)
            need = mx.flash_attn_q_workspace(s["q"], *s["kv"], s["mask"], s["out"])
            s["ws"] = torch.empty(need, dtype=torch.uint8, device=DEV)
    if case["op"] == "attn":
        return mx.flash_attn_q(s["q"], *s["kv"], s["mask"], 1.0 / math.sqrt(case["dk"]), softcap=case["softcap"], out=s["out"],
                               workspace=s["ws"])
    if case["op"] == "store":
        mx.set_rows([(s["caches"][0], s["xk"]), (s["caches"][1], s["xv"])], s["idx"])
    return mx.get_rows(s["caches"], s["idx"], torch.float16 if case.get("dst") == "F16" else torch.float32)


# ---- the definitions in 64 bits ------------------------------------------------------------

def _f32(a):
    return a.astype(np.float32).astype(np.float64)


def _stored(x, t):
    """What the rows of x [..., D] stand for once stored: the formats' own steps on the host, every
    quotient and product formed in 64 bits and rounded to the 32 (the scale to the 16) that the
    definition names."""
    b = x.cpu().numpy().astype(np.float64).reshape(-1, 32)
    i = np.arange(len(b))
    peak = b[i, np.abs(b).argmax(1)]                       # argmax: the first of equals
    d = _f32(np.abs(peak) / 127.0 if t == Q8_0 else peak / -8.0)
    inv = _f32(np.divide(1.0, d, out=np.zeros_like(d), where=d != 0))
    y = _f32(b * inv[:, None])
    if t == Q8_0:
        c = np.sign(y) * np.floor(np.abs(y) + 0.5)
    else:
        c = np.minimum(15.0, np.floor(_f32(y + 8.5))) - 8.0
    v = c * d.astype(np.float16).astype(np.float64)[:, None]
    return torch.from_numpy(v.reshape(x.shape))


def _held(planes, t):
    """The values of a cache in 64 bits."""
    codes, d = planes
    d = d.double()
    if t == Q8_0:
        return (codes.double().unflatten(-1, (-1, 32)) * d.unsqueeze(-1)).flatten(-2)
    u = codes.unflatten(-1, (-1, 16)).long()
    lo, hi = u % 16, u // 16
    return ((torch.stack([lo, hi], -2).flatten(-2) - 8) * d.unsqueeze(-1)).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "store":
        return [_stored(s["xk"], case["kt"]), _stored(s["xv"], case["vt"])]
    if case["op"] == "load":
        at = s["idx"].long()
        return [_held((c[at], d[at]), t) for (c, d), t in ((s["k"], case["kt"]), (s["v"], case["vt"]))]
    S, T, KV, H, HK, dv = (case[n] for n in ("S", "T", "KV", "H", "HK", "dv"))
    out = torch.zeros(S, T, H, dv, dtype=torch.float64, device=DEV)
    for i, n in enumerate(_lengths(case)):
        k = _held([c[i, :n] for c in s["k"]], case["kt"])
        v = _held([c[i, :n] for c in s["v"]], case["vt"])
        seen = s["mask"][i, :, :n] == 0
        for h in range(H):
            x = s["q"][i, h].double() @ k[:, h * HK // H].T.contiguous() / math.sqrt(case["dk"])
            if case["softcap"]:
                x = case["softcap"] * torch.tanh(x / case["softcap"])
            x = x.masked_fill(~seen, -math.inf)
            w = torch.exp(x - torch.logsumexp(x, -1, keepdim=True)).nan_to_num(0.0)
            out[i, :, h] = w @ v[:, h * HK // H].contiguous()
    return out

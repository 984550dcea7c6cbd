"""The operators on a KV cache in pages, as cases that can be timed and checked.

Three operators of ggml_mi355x, as a decoding step uses them one after the other:
  append  the new tokens' keys (rotated to their positions) and values stored into the pages of their
          sequences, the queries rotated in the same call; then the stored rows read back
  attend  attention of the new tokens, a chain or a tree of drafts, over the pages of their sequences
  keep    the rows of the drafts that were accepted moved to where the sequence goes on; then read back
A cache is rows [rows][heads][dim] of Q8_0, Q4_0 (planes of codes and fp16 block scales) or F16; page p is its
rows p * page and on, and a table gives each sequence's pages in order. The new tokens of a sequence
lie behind the n_past rows that it holds; some of the T places of a batch may be padding.
Head counts and dims are those of the 8B prefill, the attention tests (64, 96, 192 / 128, 256) and
the benchmark; activations are N(0, 1), as after a norm.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

Q4_0, Q8_0, F16 = "Q4_0", "Q8_0", "F16"
DEV = "cuda"


# ---- cases ---------------------------------------------------------------------------------

def listed():
    return [
        # one generated token of an 8B layer: latency counts
        dict(name="append_token_q8_0", op="append", S=1, T=1, tree=False, past=1000, page=64, H=32, HK=8, dk=128, dv=128, kt=Q8_0, vt=Q8_0, src="F32", rot=128, neox=True),
        # 24 sequences of different lengths, each with a tree of up to 16 drafts, keys in 8 bits and values in 4
        dict(name="append_trees_k8v4", op="append", S=24, T=16, tree=True, past=4000, page=32, H=32, HK=8, dk=128, dv=128, kt=Q8_0, vt=Q4_0, src="F16", rot=128, neox=True),
        # a long ragged prompt into an fp16 cache, half of each head rotated in neighbouring pairs
        dict(name="append_prompt_f16", op="append", S=1, T=4091, tree=False, past=0, page=128, H=32, HK=8, dk=128, dv=128, kt=F16, vt=F16, src="F16", rot=64, neox=False),
        # a verified tree of one sequence: five drafts stay, all 32 layers' heads in one row
        dict(name="keep_path5_q8_0", op="keep", S=1, T=16, keep=5, past=1000, page=64, HK=256, dk=128, kt=Q8_0),
        # the same for 48 sequences in 4 bits
        dict(name="keep_48seq_q4_0", op="keep", S=48, T=32, keep=9, past=700, page=32, HK=256, dk=128, kt=Q4_0),
        # one token early in a conversation
        dict(name="token_q8_0_kv1000", op="attend", S=1, T=1, tree=False, past=999, page=64, H=32, HK=8, dk=128, dv=128, kt=Q8_0, vt=Q8_0, q="F32", softcap=0.0),
        # one token deep in a long context, fp16
        dict(name="token_f16_kv32768", op="attend", S=1, T=1, tree=False, past=32767, page=128, H=32, HK=8, dk=128, dv=128, kt=F16, vt=F16, q="F16", softcap=0.0),
        # 32 sequences of different lengths served together
        dict(name="tokens_32seq_q8_0", op="attend", S=32, T=1, tree=False, past=4095, page=64, H=32, HK=8, dk=128, dv=128, kt=Q8_0, vt=Q8_0, q="F16", softcap=0.0),
        # a tree of 16 drafts to verify, heads of 256 with a soft-cap
        dict(name="tree16_k8v4_d256", op="attend", S=1, T=16, tree=True, past=16001, page=32, H=16, HK=8, dk=256, dv=256, kt=Q8_0, vt=Q4_0, q="F32", softcap=50.0),
        # ten sequences with trees of up to 64 drafts each, fp16, a small model's heads
        dict(name="trees64_f16_d64", op="attend", S=10, T=64, tree=True, past=3001, page=256, H=32, HK=8, dk=64, dv=64, kt=F16, vt=F16, q="F16", softcap=0.0),
        # a very long context in 4 bits, five drafts
        dict(name="tree5_q4_0_kv131072", op="attend", S=1, T=5, tree=True, past=131067, page=256, H=32, HK=8, dk=128, dv=128, kt=Q4_0, vt=Q4_0, q="F32", softcap=0.0),
        # a micro-batch of a prompt deep in its context
        dict(name="chunk512_q8_0_kv8192", op="attend", S=1, T=512, tree=False, past=7680, page=64, H=32, HK=8, dk=128, dv=128, kt=Q8_0, vt=Q8_0, q="F32", softcap=0.0),
    ]


def _log(rng, lo, hi):
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "append", "keep", "attend", "attend", "attend", "attend"])
    page = rng.choice([32, 64, 96, 128, 256])
    kt, vt = rng.choice([(Q8_0, Q8_0), (Q4_0, Q4_0), (Q8_0, Q4_0), (Q4_0, Q8_0), (F16, F16)])
    dk, dv, H, HK = rng.choice([(64, 64, 32, 8), (96, 96, 16, 16), (128, 128, 32, 8), (128, 128, 32, 4), (128, 128, 16, 16),
                                (192, 128, 16, 16), (256, 256, 16, 8)])
    S = rng.choice([1, 1, _log(rng, 2, 48)])
    if op == "keep":
        T = _log(rng, 2, 64)
        return dict(op=op, S=S, T=T, keep=rng.randint(1, min(T, 16)), past=_log(rng, 1, 4096), page=page, HK=rng.choice([8, 64, 256]),
                    dk=rng.choice([64, 96, 128]), kt=rng.choice([Q8_0, Q4_0, F16]))
    tree = rng.random() < 0.5
    if op == "append":
        T = _log(rng, 2, 64) if tree else _log(rng, 1, max(1, 4091 // S))
        T = min(T, 4091 * 32 * 128 // (S * H * dk))
        return dict(op=op, S=S, T=T, tree=tree, past=rng.choice([0, _log(rng, 1, 100000 // S)]), page=page, H=H, HK=HK, dk=dk, dv=dv, kt=kt, vt=vt,
                    src=rng.choice(["F32", "F16"]), rot=rng.choice([dk, dk // 2]), neox=rng.random() < 0.5)
    T = _log(rng, 2, 64) if tree else rng.choice([1, 1, _log(rng, 2, 512) if S == 1 else _log(rng, 2, 32)])
    # rows held, and pairs of rows, as many as in the largest listed cases
    most = min(131072 * 8 * 256 // (S * HK * (dk + dv)), 512 * 8192 * 32 * 256 // (S * T * H * (dk + dv)), 131072)
    return dict(op=op, S=S, T=T, tree=tree, past=rng.choice([0, _log(rng, 1, most), _log(rng, 1, most)]) if tree else _log(rng, 1, most), page=page,
                H=H, HK=HK, dk=dk, dv=dv, kt=kt, vt=vt, q=rng.choice(["F32", "F16"]), softcap=rng.choice([0.0, 0.0, 0.0, 50.0]))


def _held(case):
    """(n_past, n_new) of each sequence: all of both for one, spread over (0, past] and (0, T] for several."""
    S, past, T = case["S"], case["past"], case["T"]
    if S == 1:
        return [past], [T]
    least = case.get("keep", 1)
    return ([round(past * (1 - (0.618034 * s) % 1.0)) for s in range(S)],
            [max(least, round(T * (1 - (0.414214 * s) % 1.0))) for s in range(S)])


def _parents(case):
    """parent[s][t] of each new token; None for a chain. Node t hangs on the root or a node shortly before it."""
    if not case.get("tree"):
        return None
    t = np.arange(case["T"])
    return np.stack([np.where(t < 2 + s % 3, -1, np.maximum(0, (t - 2) // 2 - (5 * t + s) % 3)) for s in range(case["S"])]).astype(np.int32)


def _bits(t):
    return {Q8_0: 8.5, Q4_0: 4.5, F16: 16.0, "F32": 32.0}[t]


def work(case):
    HK, dk = case["HK"], case["dk"]
    past, new = _held(case)
    tokens = sum(new)
    if case["op"] == "keep":     # rows read and written, and read back with their values out
        moved = case["S"] * case["keep"] * HK * dk
        return {"bytes": moved * (3 * _bits(case["kt"]) / 8 + 2), "flops": 1.0 * moved}
    H, dv = case["H"], case["dv"]
    held = (dk * _bits(case["kt"]) + dv * _bits(case["vt"])) / 8      # bytes of one position of one KV head
    if case["op"] == "append":   # sources in, rotated queries out, rows written and read, their values out
        src = _bits(case["src"]) / 8
        return {"bytes": tokens * (HK * ((dk + dv) * (src + 2) + 2 * held) + H * dk * 2 * src),
                "flops": 3.0 * tokens * ((H + HK) * case["rot"] + HK * (dk + dv))}
    pairs = 0
    parents = _parents(case)
    for s in range(case["S"]):
        depth = []
        for t in range(new[s]):
            up = t - 1 if parents is None else int(parents[s][t])
            depth.append(1 if up < 0 else depth[up] + 1)
        pairs += past[s] * new[s] + sum(depth)
    return {"bytes": tokens * H * (dk * _bits(case["q"]) / 8 + dv * 2) + (sum(past) + tokens) * HK * held, "flops": 2.0 * pairs * H * (dk + dv)}


# ---- inputs --------------------------------------------------------------------------------

def _random_cache(g, t, *shape):
    """(codes, scales) of a cache holding N(0, 1) values, every block scaled to its largest; F16: (values,)."""
    x = torch.randn(*shape[:-1], shape[-1] // 32, 32, generator=g, device=DEV)
    if t == F16:
        return (x.half().reshape(*shape),)
    d = (x.abs().amax(-1, keepdim=True) / (127.0 if t == Q8_0 else 8.0)).half()
    x = x.div_(d.float()).round_()
    if t == Q8_0:
        return x.clamp_(-127, 127).to(torch.int8).reshape(*shape), d.squeeze(-1)
    u = x.clamp_(-8, 7).add_(8).to(torch.uint8)
    return (u[..., :16] | (u[..., 16:] << 4)).reshape(*shape[:-1], shape[-1] // 2), d.squeeze(-1)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    S, T, page, HK, dk = (case[n] for n in ("S", "T", "page", "HK", "dk"))
    past, new = _held(case)
    n_table = (max(p + n for p, n in zip(past, new)) + page - 1) // page + 1
    used = [(p + n + page - 1) // page for p, n in zip(past, new)]
    pages = sum(used) + 3
    # the pool's pages in no order, each sequence's own; entries behind a sequence's last page name no page
    order, at = torch.randperm(pages, generator=g, device=DEV).int(), 0
    table = torch.full((S, n_table), -1, dtype=torch.int32, device=DEV)
    for s in range(S):
        table[s, :used[s]] = order[at:at + used[s]]
        at += used[s]
    parents = _parents(case)
    s = dict(case=dict(case), table=table, n_past=torch.tensor(past, dtype=torch.int32, device=DEV),
             n_new=torch.tensor(new, dtype=torch.int32, device=DEV),
             parents=None if parents is None else torch.from_numpy(parents).to(DEV), max_kv=max(p + n for p, n in zip(past, new)))
    s["k"] = _random_cache(g, case["kt"], pages * page, HK, dk)
    real = torch.arange(T, device=DEV)[None, :] < s["n_new"][:, None]
    j = s["n_past"][:, None].long() + torch.arange(T, device=DEV)[None, :]
    j = j.clamp(max=n_table * page - 1)
    rows = table.gather(1, j // page).long() * page + j % page           # [S][T] rows of the new tokens
    if case["op"] == "keep":
        # paths as a tree numbered level by level gives them: drafts in place first, the others from behind the kept rows
        keep = case["keep"]
        path = np.zeros((S, keep), np.int32)
        for i in range(S):
            stay = min(keep, i % 3)
            if new[i] - keep < keep - stay:
                stay = keep - max(0, new[i] - keep)
            step = (new[i] - keep) // max(1, keep - stay)
            path[i] = [a if a < stay else keep + (a - stay) * max(1, step) for a in range(keep)]
        s["path"] = torch.from_numpy(path).to(DEV)
        s["rows"] = rows
        s["idx"] = rows[:, :keep].reshape(-1).int()
        return s
    s["v"] = _random_cache(g, case["vt"], pages * page, HK, case["dv"])
    H = case["H"]
    src = torch.float16 if case.get("src", case.get("q")) == "F16" else torch.float32
    q = torch.randn(S, T, H, dk, generator=g, device=DEV).to(src)
    if case["op"] == "attend":
        s["q"] = q
        return s
    s["xq"] = q
    s["xk"] = torch.randn(S, T, HK, dk, generator=g, device=DEV).to(src)
    s["xv"] = torch.randn(S, T, HK, case["dv"], generator=g, device=DEV).to(src)
    rot = case["rot"]
    s["freq"] = (500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).float().to(DEV)
    s["q_out"] = torch.zeros_like(q)
    s["idx"], s["at"] = rows[real].int(), real.nonzero(as_tuple=True)
    return s


# ---- one pass ------------------------------------------------------------------------------

def _plain_codes(x, t):
    """The codes and scales of x [..., D] by the formats' definition: a block's scale is max|x| / 127
    (Q8_0) or the value of largest magnitude (the first of equals) / -8 (Q4_0), codes are x times the
    reciprocal of the scale, rounded half away from zero. Each product and quotient is a 32-bit one;
    they are formed in 64 bits and rounded, since a value next to a border changes its code."""
    if t == F16:
        return (x.half(),)
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


def _plain_values(planes, t):
    if t == F16:
        return planes[0].float()
    codes, d = planes
    if t == Q8_0:
        c = codes.float().reshape(*d.shape, 32)
    else:
        u = codes.reshape(*d.shape, 16)
        c = torch.cat([u & 15, u >> 4], -1).float() - 8.0
    return (c * d.float()[..., None]).flatten(-2)


def _seen(s):
    """[S][T][T]: whether a new token sees another, itself among them; padding sees nothing."""
    case = s["case"]
    S, T = case["S"], case["T"]
    real = torch.arange(T, device=DEV)[None, :] < s["n_new"][:, None]
    if s["parents"] is None:
        reach = torch.ones(T, T, device=DEV).tril()[None].expand(S, T, T)
    else:
        # one step up is a matrix; its powers with the unit matrix count the ways up
        up = torch.eye(T + 1, dtype=torch.float64, device=DEV)[s["parents"].long() % (T + 1)][..., :T]
        reach = torch.linalg.matrix_power(up + torch.eye(T, dtype=torch.float64, device=DEV), T)
    return (reach > 0) & real[:, :, None] & real[:, None, :]


def _plain_append(s):
    case = s["case"]
    rot, T = case["rot"], case["T"]
    at, idx = s["at"], s["idx"].long()
    depth = torch.arange(T, device=DEV)[None, :].expand(case["S"], T) if s["parents"] is None else _seen(s).sum(-1) - 1
    pos = (s["n_past"][:, None] + depth).double()[at]
    a = pos[:, None] * s["freq"].double()                      # far positions: in 64 bits
    c, n = a.cos().float().double()[:, None, :], a.sin().float().double()[:, None, :]

    def turned(x):     # every product and sum a 32-bit one, as if formed in 64 and rounded
        y = x.float().clone()
        x = x.double()
        i, j = (slice(0, rot // 2), slice(rot // 2, rot)) if case["neox"] else (slice(0, rot, 2), slice(1, rot, 2))
        y[..., i] = ((x[..., i] * c).float().double() - (x[..., j] * n).float().double()).float()
        y[..., j] = ((x[..., i] * n).float().double() + (x[..., j] * c).float().double()).float()
        return y

    s["q_out"][at] = turned(s["xq"][at]).to(s["q_out"].dtype)
    for planes, x, t in ((s["k"], turned(s["xk"][at]), case["kt"]), (s["v"], s["xv"][at].float(), case["vt"])):
        for p, new in zip(planes, _plain_codes(x, t)):
            p[idx] = new
    return [s["q_out"]] + [_plain_values([p[idx] for p in planes], t).half() for planes, t in ((s["k"], case["kt"]), (s["v"], case["vt"]))]


def _plain_keep(s):
    case = s["case"]
    src, idx = s["rows"].gather(1, s["path"].long()).reshape(-1), s["idx"].long()
    for p in s["k"]:
        p[idx] = p[src]
    return _plain_values([p[idx] for p in s["k"]], case["kt"]).half()


def _plain_attend(s):
    case = s["case"]
    S, T, H, HK, dk, dv, page = (case[n] for n in ("S", "T", "H", "HK", "dk", "dv", "page"))
    j = torch.arange(s["max_kv"], device=DEV)
    n_past, n_new = s["n_past"].long()[:, None], s["n_new"].long()[:, None]
    here = j[None, :] < n_past + n_new
    rows = torch.where(here, s["table"][:, j // page].long() * page + j % page, 0)
    k = _plain_values([p[rows] for p in s["k"]], case["kt"]).transpose(1, 2).contiguous()        # [S][HK][KV][dk]
    v = _plain_values([p[rows] for p in s["v"]], case["vt"]).transpose(1, 2).contiguous()
    q = s["q"].float().transpose(1, 2).reshape(S, HK, H // HK * T, dk)
    p = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(1.0 / math.sqrt(dk)).view(S, H, T, -1)
    if case["softcap"]:
        p = p.div_(case["softcap"]).tanh_().mul_(case["softcap"])
    u = (j[None, :] - n_past).clamp(0, T - 1)
    see = _seen(s).gather(2, u[:, None, :].expand(S, T, -1))
    see = torch.where((j[None, :] < n_past)[:, None, :], (torch.arange(T, device=DEV)[None, :] < n_new)[:, :, None], see & here[:, None, :])
    p = p.masked_fill_(~see[:, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    den = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(S, HK, H // HK * T, -1), v).view(S, H, T, dv)
    return torch.where(den > 0, o / den, 0.0).transpose(1, 2).contiguous().half()


def _mx():
    at = os.path.join(os.getcwd(), "ggml-rocket_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import ggml_mi355x
    return ggml_mi355x


def run(s):
    case = s["case"]
    if not own:
        return {"append": _plain_append, "keep": _plain_keep, "attend": _plain_attend}[case["op"]](s)
    mx = _mx()
    if "step" not in s:      # a program keeps its caches, the step's description, its workspace and its output buffers
        kind = {Q8_0: mx.Q8_0, Q4_0: mx.Q4_0, F16: mx.F16}
        s["caches"] = [mx.KvCache(kind[case[t]], *s[n]) for n, t in (("k", "kt"), ("v", "vt")) if n in s]
        s["step"] = mx.KvStep(s["table"], s["n_past"], case["T"], case["page"], n_new=s["n_new"], parents=s["parents"])
        if case["op"] == "append":
            s["rope"] = mx.Rope(s["freq"], neox=case["neox"])
        if case["op"] == "attend":
            s["out"] = torch.empty(case["S"], case["T"], case["H"], case["dv"], dtype=torch.float16, device=DEV)
            s["qv"] = s["q"].permute(0, 2, 1, 3)
            need = mx.flash_attn_paged_workspace(s["qv"], *s["caches"], s["step"], s["out"], max_kv=s["max_kv"])
            s["ws"] = torch.empty(need, dtype=torch.uint8, device=DEV)
    if case["op"] == "attend":
        return mx.flash_attn_paged(s["qv"], *s["caches"], s["step"], 1.0 / math.sqrt(case["dk"]), softcap=case["softcap"], out=s["out"],
                                   workspace=s["ws"], max_kv=s["max_kv"])
    if case["op"] == "keep":
        mx.kv_keep(s["step"], s["caches"], s["path"])
        return mx.get_rows(s["caches"], s["idx"], torch.float16)[0]
    mx.kv_append(s["step"], *s["caches"], s["xk"], s["xv"], rope=s["rope"], q=s["xq"], q_out=s["q_out"])
    return [s["q_out"]] + mx.get_rows(s["caches"], s["idx"], torch.float16)


# ---- the definitions in 64 bits ------------------------------------------------------------

def _f32(a):
    return a.astype(np.float32).astype(np.float64)


def _stored(x, t):
    """What the rows of x [..., D] (64-bit values that 32 bits hold) stand for once stored: the formats' own
    steps on the host, every quotient and product formed in 64 bits and rounded to the 32 (the scale
    to the 16) that the definition names."""
    if t == F16:
        return x.astype(np.float16).astype(np.float64)
    b = x.reshape(-1, 32)
    i = np.arange(len(b))
    peak = b[i, np.abs(b).argmax(1)]                       # argmax: the first of equals
    d = _f32(np.abs(peak) / 127.0 if t == Q8_0 else peak / -8.0)
    inv = _f32(np.divide(1.0, d, out=np.zeros_like(d), where=d != 0))
    y = _f32(b * inv[:, None])
    if t == Q8_0:
        c = np.sign(y) * np.floor(np.abs(y) + 0.5)
    else:
        c = np.minimum(15.0, np.floor(_f32(y + 8.5))) - 8.0
    return (c * d.astype(np.float16).astype(np.float64)[:, None]).reshape(x.shape)


def _cache_values(planes, t):
    """The values of cache rows in 64 bits."""
    if t == F16:
        return planes[0].double()
    codes, d = planes
    d = d.double()
    if t == Q8_0:
        return (codes.double().unflatten(-1, (-1, 32)) * d.unsqueeze(-1)).flatten(-2)
    u = codes.unflatten(-1, (-1, 16)).long()
    lo, hi = u % 16, u // 16
    return ((torch.stack([lo, hi], -2).flatten(-2) - 8) * d.unsqueeze(-1)).flatten(-2)


def _chains(case):
    """For each sequence and new token the new tokens on its way up, itself first."""
    parents, new = _parents(case), _held(case)[1]
    found = []
    for s in range(case["S"]):
        ways = []
        for t in range(new[s]):
            up = t - 1 if parents is None else int(parents[s][t])
            ways.append([t] + (ways[up] if up >= 0 else []))
        found.append(ways)
    return found


def _exact_append(case, s):
    past, new = _held(case)
    rot, out, rows = case["rot"], [], {"k": [], "v": []}
    parents = _parents(case)
    freq = s["freq"].cpu().numpy().astype(np.float64)
    q_out = np.zeros(tuple(s["xq"].shape))
    xq, xk, xv = (s[n].cpu().numpy().astype(np.float64) for n in ("xq", "xk", "xv"))
    even = np.arange(rot // 2) if case["neox"] else np.arange(0, rot, 2)
    odd = even + (rot // 2 if case["neox"] else 1)
    for i in range(case["S"]):
        level = np.arange(new[i]) if parents is None else np.array([len(w) - 1 for w in _chains(case)[i]])
        a = (past[i] + level).astype(np.float64)[:, None, None] * freq
        c, n = _f32(np.cos(a)), _f32(np.sin(a))

        def turned(x):
            y = x.copy()
            y[..., even] = _f32(_f32(x[..., even] * c) - _f32(x[..., odd] * n))
            y[..., odd] = _f32(_f32(x[..., even] * n) + _f32(x[..., odd] * c))
            return y

        q_out[i, :new[i]] = turned(xq[i, :new[i]])
        rows["k"].append(_stored(turned(xk[i, :new[i]]), case["kt"]))
        rows["v"].append(_stored(xv[i, :new[i]], case["vt"]))
    return [torch.from_numpy(q_out)] + [torch.from_numpy(np.concatenate(rows[n])) for n in ("k", "v")]


def _exact_keep(case, s):
    out = []
    path, table, page = s["path"].tolist(), s["table"].tolist(), case["page"]
    for i, n in enumerate(_held(case)[0]):
        for u in path[i]:
            row = table[i][(n + u) // page] * page + (n + u) % page
            out.append(_cache_values([p[row] for p in s["k"]], case["kt"]))
    return torch.stack(out)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, s)
    if case["op"] == "keep":
        return _exact_keep(case, s)
    S, T, H, HK, dv, page = (case[n] for n in ("S", "T", "H", "HK", "dv", "page"))
    out = torch.zeros(S, T, H, dv, dtype=torch.float64, device=DEV)
    past, new = _held(case)
    ways = _chains(case)
    for i in range(S):
        n = past[i] + new[i]
        rows = torch.cat([torch.arange(p * page, (p + 1) * page, device=DEV) for p in s["table"][i, :(n + page - 1) // page].tolist()])[:n]
        hide = np.zeros((new[i], n), bool)
        hide[:, past[i]:] = True
        for t, way in enumerate(ways[i]):
            hide[t, [past[i] + u for u in way]] = False
        hide = torch.from_numpy(hide).to(DEV)
        for hk in range(HK):
            k = _cache_values([p[rows, hk] for p in s["k"]], case["kt"])
            v = _cache_values([p[rows, hk] for p in s["v"]], case["vt"])
            for h in range(hk * H // HK, (hk + 1) * H // HK):
                x = s["q"][i, :new[i], h].double() @ k.T.contiguous() / math.sqrt(case["dk"])
                if case["softcap"]:
                    x = case["softcap"] * torch.tanh(x / case["softcap"])
                x = x.masked_fill(hide, -math.inf)
                out[i, :new[i], h] = torch.exp(x - torch.logsumexp(x, -1, keepdim=True)) @ v
    return out

"""Operators of a shared and of a shrinking key-value cache, as they are measured.

* ``append``  norms of queries and keys per head, rotary positions and the append in one pass
* ``prefix``  one new token per sequence, the sequences beginning with the same pages
* ``mass``    attention weight that each slot of the cache has received, added up
* ``evict``   the slots of least weight leave the cache

Activations are f32, caches fp16, bf16 or e4m3 (with one scale each for keys and values).
``own`` selects the framework's kernels; otherwise ``run`` is the plain torch form.
"""
import math
import random

import numpy as np
import torch

own = False

CACHE = {"f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
SCALES = {"f16": (1.0, 1.0), "bf16": (1.0, 1.0), "e4m3": (0.03125, 0.0234375)}   # of keys, of values
EPS = 1e-6


def listed():
    return [
        # a single user's token entering the cache: latency only
        dict(name="append one token", op="append", tokens=1, seqs=1, hi=1000, hq=32, hkv=8, d=128,
             rot=128, pairs="half", cache="f16", page=16, gemma=False, ledger=False),
        # one decode step of a batch whose caches have been shrunk: slots apart from positions,
        # weights around 1, 8-bit cache
        dict(name="append decode batch", op="append", tokens=64, seqs=64, hi=2048, hq=16, hkv=8,
             d=256, rot=128, pairs="adjacent", cache="e4m3", page=32, gemma=True, ledger=True),
        # prompts of five sequences entering together
        dict(name="append prompts", op="append", tokens=8191, seqs=5, hi=4096, hq=32, hkv=8, d=128,
             rot=128, pairs="half", cache="bf16", page=16, gemma=False, ledger=False),
        # a few samples of one short prompt: latency
        dict(name="prefix few short", op="prefix", seqs=4, prefix=512, lo=1, hi=64, hq=32, hkv=8,
             d=128, cache="f16", page=16, cap=0.0),
        # a serving batch behind a long system prompt, empty rows among it
        dict(name="prefix batch", op="prefix", seqs=64, prefix=8192, lo=0, hi=1024, hq=32, hkv=8,
             d=128, cache="f16", page=16, cap=0.0),
        # many questions about one long document
        dict(name="prefix document", op="prefix", seqs=256, prefix=32768, lo=1, hi=300, hq=32,
             hkv=8, d=128, cache="bf16", page=64, cap=0.0),
        # wide heads, capped scores, rows that fill no tile
        dict(name="prefix wide heads", op="prefix", seqs=37, prefix=6000, lo=0, hi=500, hq=16,
             hkv=4, d=256, cache="f16", page=24, cap=50.0),
        # 8-bit cache, three query heads to a key head
        dict(name="prefix 8-bit", op="prefix", seqs=100, prefix=16384, lo=1, hi=700, hq=24, hkv=8,
             d=128, cache="e4m3", page=32, cap=0.0),
        # a chat's weights, step by step
        dict(name="mass one short", op="mass", seqs=1, lo=333, hi=333, hq=32, hkv=8, d=128,
             cache="f16", page=16, cap=0.0),
        # a serving batch of ragged lengths
        dict(name="mass batch", op="mass", seqs=64, lo=0, hi=4096, hq=32, hkv=8, d=128,
             cache="bf16", page=16, cap=0.0),
        # every step of a batch at its limit: one slot of each sequence and head leaves
        dict(name="evict one each", op="evict", seqs=128, lo=1025, hi=1025, keep=1024, recent=128,
             hkv=8, d=128, cache="bf16", page=16),
        # long prompts shrunk before the first answer
        dict(name="evict prompts", op="evict", seqs=6, lo=20000, hi=32768, keep=4096, recent=1024,
             hkv=8, d=128, cache="f16", page=16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "prefix", "prefix", "mass", "evict"])
    d = rng.choice([64, 80, 96, 128, 128, 192, 256])
    hkv = rng.choice([1, 2, 4, 8, 8, 16])
    hq = hkv * rng.choice([1, 2, 3, 4, 5, 8]) if hkv < 16 else hkv * rng.choice([1, 2])
    cache = rng.choice(["f16", "bf16", "e4m3"])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    if op == "append":
        tokens = _log(rng, 1, max(2, min(8192, (1 << 25) // ((hq + 2 * hkv) * d))))
        decode = rng.random() < 0.5 and tokens <= 512
        return dict(op=op, tokens=tokens, seqs=tokens if decode else rng.randint(1, min(tokens, 16)),
                    hi=_log(rng, 16, max(17, min(65536, (1 << 27) // (tokens * hkv * d)))) if decode
                    else max(64, tokens), hq=hq, hkv=hkv, d=d,
                    rot=rng.choice([d, d, d // 2]), pairs=rng.choice(["half", "adjacent"]),
                    cache=cache, page=page, gemma=rng.random() < 0.5, ledger=decode)
    if op == "prefix":
        seqs = _log(rng, 2, 256)
        most = min(32768, (1 << 35) // (seqs * hq * d))     # a quarter of the largest case's work
        own_hi = _log(rng, 1, max(2, min(2048, (1 << 26) // (seqs * hkv * d))))
        return dict(op=op, seqs=seqs, prefix=page * max(1, _log(rng, 16, max(17, most)) // page),
                    lo=rng.choice([0, 1, own_hi]), hi=own_hi, hq=hq, hkv=hkv, d=d, cache=cache,
                    page=page, cap=rng.choice([0.0, 0.0, 30.0]))
    keys = (1 << 26) // (hkv * d)                           # of the whole batch, at most
    seqs = _log(rng, 1, 256)
    hi = _log(rng, 16, max(17, min(65536, keys // seqs)))
    lo = rng.choice([0, 1, hi // 2, hi])
    if op == "mass":
        return dict(op=op, seqs=seqs, lo=lo, hi=hi, hq=hq, hkv=hkv, d=d, cache=cache, page=page,
                    cap=rng.choice([0.0, 0.0, 30.0]))
    keep = rng.choice([max(1, hi - 1), max(1, hi // 2), max(1, hi // 9)])
    return dict(op=op, seqs=seqs, lo=lo, hi=hi, keep=keep, recent=rng.choice([0, keep // 4, keep]),
                hkv=hkv, d=d, cache=cache, page=page)


def _lens(case):
    """Keys of each sequence (of its own, behind a prefix): the case's own, whatever the seed."""
    r = random.Random(case["seqs"] * 1000003 + case["hi"])
    lens = [r.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]
    lens[r.randrange(len(lens))] = case["hi"]
    if case["op"] == "prefix":                     # a row without own keys is padding
        lens = [n + case["prefix"] if n else 0 for n in lens]
    return lens


def _spread(case):
    """(sequence, slot) of every token of an append case."""
    r = random.Random(case["tokens"] * 1000003 + case["hi"])
    T, S = case["tokens"], case["seqs"]
    if S == T:                                     # one new token each
        return list(range(T)), [r.randrange(case["hi"]) for _ in range(T)]
    cuts = sorted(r.sample(range(1, T), S - 1)) if S > 1 else []
    seq, pos = [], []
    for s, (a, b) in enumerate(zip([0] + cuts, cuts + [T])):
        seq += [s] * (b - a)
        pos += range(b - a)
    return seq, pos


def work(case):
    hkv, d = case["hkv"], case["d"]
    e = 1 if case["cache"] == "e4m3" else 2
    if case["op"] == "append":
        T, hq = case["tokens"], case["hq"]
        return {"bytes": T * ((2 * hq + 2 * hkv) * d * 4 + 2 * hkv * d * e
                              + (8 * hkv if case["ledger"] else 0)),
                "flops": T * (hq + hkv) * (3 * d + 3 * case["rot"])}
    lens = _lens(case)
    if case["op"] == "prefix":
        S, hq, P = case["seqs"], case["hq"], case["prefix"]
        own_keys = sum(n - P for n in lens if n)
        return {"bytes": 2 * (P + own_keys) * hkv * d * e + S * hq * (2 * d + 1) * 4,
                "flops": 4 * sum(lens) * hq * d}
    if case["op"] == "mass":
        return {"bytes": sum(lens) * hkv * (d * e + 8) + case["seqs"] * case["hq"] * (d + 1) * 4,
                "flops": 2 * sum(lens) * case["hq"] * d}
    # survivors are spread evenly but for the recent ones: what lies behind `keep` moves
    keep = case["keep"]
    moved = sum(keep * (n - keep) // n for n in lens if n > keep)
    return {"bytes": hkv * (sum(8 * n + 8 * min(n, keep) for n in lens) + 4 * moved * d * e),
            "flops": hkv * sum(lens)}


# ------------------------------------------------------------------- inputs

def _pool(case, total, g):
    shape = (total, case["page"], case["hkv"], case["d"])
    caches = []
    for scale in SCALES[case["cache"]]:
        c = torch.empty(shape, dtype=CACHE[case["cache"]], device="cuda")
        for at in range(0, total, 4096):
            part = torch.randn((min(4096, total - at),) + shape[1:], generator=g, device="cuda")
            c[at:at + 4096].copy_(part / scale)
        caches.append(c)
    return caches


def _pages(case, need, g, shared=0):
    """Caches of a pool with a few pages more than needed, and the page table: `shared` pages at
    the front of every row that has any, then pages of its own; -1 behind a sequence's last page."""
    mine = [max(0, n - shared) for n in need]
    total, width = shared + sum(mine) + 3, max(need) + 1
    caches = _pool(case, total, g)
    free = torch.randperm(total, generator=g, device="cuda", dtype=torch.int32)
    counts = torch.tensor(mine, device="cuda")
    first = torch.cumsum(counts, 0) - counts + shared
    col = torch.arange(width, device="cuda")
    at = torch.where(col < shared, col, first[:, None] + col - shared).clamp(max=total - 1)
    held = torch.tensor(need, device="cuda")[:, None]
    return caches, torch.where(col < held, free[at], -1).to(torch.int32).contiguous(), free[:shared]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    st = {"case": case}
    if own:
        from linuxnightmaresuite_b200 import kernels
        st["K"] = kernels
    hkv, d, page = case["hkv"], case["d"], case["page"]
    if case["op"] == "append":
        hq, T = case["hq"], case["tokens"]
        seq, slot = _spread(case)
        last = [0] * case["seqs"]
        for s, p in zip(seq, slot):
            last[s] = max(last[s], p)
        (st["k_cache"], st["v_cache"]), st["table"], _ = _pages(
            case, [p // page + 1 for p in last], g)
        st["slots"] = torch.tensor(slot, dtype=torch.int32, device="cuda")
        st["seq_ids"] = None if case["seqs"] == T else torch.tensor(
            seq, dtype=torch.int32, device="cuda")
        st["positions"] = st["slots"]
        if case["ledger"]:                         # tokens have left: positions run ahead of slots
            st["positions"] = st["slots"] + torch.randint(0, 60000, (T,), generator=g,
                                                          device="cuda", dtype=torch.int32)
            shape = (case["seqs"], hkv, max(last) + 1)
            st["mass"] = torch.rand(shape, generator=g, device="cuda")
            st["held"] = torch.randint(0, 1 << 20, shape, generator=g, device="cuda",
                                       dtype=torch.int32)
        i = torch.arange(case["rot"] // 2, dtype=torch.float64, device="cuda")
        st["inv_freq"] = 10000.0 ** (-2.0 * i / case["rot"])
        st["wq"], st["wk"] = (0.1 * torch.randn(d, generator=g, device="cuda")
                              + (0.0 if case["gemma"] else 1.0) for _ in range(2))
        # as the joint projection leaves them: q, k, v of a token side by side
        qkv = 2.0 * torch.randn((T, (hq + 2 * hkv) * d), generator=g, device="cuda")
        st["q"] = qkv[:, :hq * d].unflatten(1, (hq, d))
        st["k"] = qkv[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
        st["v"] = qkv[:, (hq + hkv) * d:].unflatten(1, (hkv, d))
        return st
    lens = _lens(case)
    shared = case["prefix"] // page if case["op"] == "prefix" else 0
    (st["k_cache"], st["v_cache"]), st["table"], st["prefix_pages"] = _pages(
        case, [-(-n // page) for n in lens], g, shared)
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    st["longest"] = max(lens)
    S = case["seqs"]
    if case["op"] == "evict":
        shape = (S, hkv, st["longest"])
        # a few slots hold most of the weight, some have received none
        m = torch.randn(shape, generator=g, device="cuda").mul_(2.0).exp_()
        st["mass"] = torch.where(torch.rand(shape, generator=g, device="cuda") < 0.02, 0.0, m)
        order = torch.rand(shape, generator=g, device="cuda").argsort(-1)
        st["held"] = (3 * order + 17).to(torch.int32)
        st["mass_out"] = torch.zeros((S, hkv, case["keep"]), device="cuda")
        st["held_out"] = torch.zeros((S, hkv, case["keep"]), dtype=torch.int32, device="cuda")
        st["lens_out"] = torch.zeros(S, dtype=torch.int32, device="cuda")
        return st
    hq = case["hq"]
    st["q"] = 1.5 * torch.randn((S, hq, d), generator=g, device="cuda")
    if case["op"] == "prefix":
        if own:
            st["ws"] = kernels.prefix_attention_workspace(S, hq, hkv, d, "cuda")
        return st
    st["mass"] = 3.0 * torch.rand((S, hkv, st["longest"]), generator=g, device="cuda")
    st["mass_out"] = torch.zeros_like(st["mass"])
    # as the attention leaves it
    st["lse"] = torch.full((S, hq), -math.inf, device="cuda")
    for s in range(S):
        if lens[s]:
            st["lse"][s] = torch.logsumexp(_scores(st, s, lens[s]), -1).flatten()
    return st


# ------------------------------------------------------------------- one pass

def _append_plain(st):
    case, q, k, v = st["case"], st["q"], st["k"], st["v"]
    h = case["rot"] // 2
    angle = st["positions"].double()[:, None, None] * st["inv_freq"]
    cos, sin = angle.cos().float(), angle.sin().float()

    def turn(x, w):
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * (1.0 + w if case["gemma"] else w)
        r, rest = x[..., :2 * h], x[..., 2 * h:]
        if case["pairs"] == "half":
            a, b = r[..., :h], r[..., h:]
            return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
        a, b = r[..., 0::2], r[..., 1::2]
        return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)

    at = st["slots"].long()
    rows = st["seq_ids"].long() if st["seq_ids"] is not None else torch.arange(len(at), device="cuda")
    page = st["table"][rows, at // case["page"]].long()
    slot = at % case["page"]
    for x, c, scale in ((turn(k, st["wk"]), st["k_cache"], SCALES[case["cache"]][0]),
                        (v, st["v_cache"], SCALES[case["cache"]][1])):
        if case["cache"] == "e4m3":
            c.view(torch.uint8)[page, slot] = (x / scale).clamp(-448, 448).to(c.dtype).view(torch.uint8)
        else:
            c[page, slot] = x.to(c.dtype)
    if not case["ledger"]:
        return turn(q, st["wq"]), st["k_cache"], st["v_cache"]
    st["mass"][rows, :, at] = 0.0
    st["held"][rows, :, at] = st["positions"][:, None]
    return turn(q, st["wq"]), st["k_cache"], st["v_cache"], st["mass"], st["held"]


def _scores(st, s, n):
    """(hkv, group, n) of sequence s."""
    case = st["case"]
    hkv, d, page = case["hkv"], case["d"], case["page"]
    k = st["k_cache"][st["table"][s, :-(-n // page)].long()].flatten(0, 1)[:n].float()
    z = st["q"][s].view(hkv, -1, d) @ (k * SCALES[case["cache"]][0]).permute(1, 2, 0)
    z = z * (1.0 / math.sqrt(d))
    return case["cap"] * torch.tanh(z / case["cap"]) if case["cap"] else z


def _prefix_plain(st):
    case, q, page = st["case"], st["q"], st["case"]["page"]
    S, hq, d = q.shape
    hkv, P = case["hkv"], case["prefix"]
    ks, vs = SCALES[case["cache"]]
    qg = q.view(S, hkv, hq // hkv, d) * (1.0 / math.sqrt(d))
    # the prefix: one product for the rows of all sequences
    pages = st["prefix_pages"].long()
    kp, vp = (c[pages].flatten(0, 1).transpose(0, 1).float() * x
              for c, x in ((st["k_cache"], ks), (st["v_cache"], vs)))          # (hkv, P, d)
    # each sequence's own tokens
    L = max(st["longest"] - P, 1)
    t = P + torch.arange(L, device="cuda")
    seen = t < st["lens"].long()[:, None]
    t = torch.where(seen, t, P)
    own_pages = st["table"].long().gather(1, t // page).clamp(min=0)
    ko = st["k_cache"][own_pages, t % page].float() * ks                       # (S, L, hkv, d)
    vo = st["v_cache"][own_pages, t % page].float() * vs
    live = (st["lens"] > 0)[:, None, None]
    out = torch.empty_like(q).view(S, hkv, -1, d)
    lse = torch.empty(qg.shape[:3], device="cuda")
    for h in range(hkv):
        rows = qg[:, h].reshape(-1, d)
        z0 = (rows @ kp[h].t()).view(S, -1, P)
        z1 = qg[:, h] @ ko[:, :, h].transpose(1, 2)
        if case["cap"]:
            z0 = case["cap"] * torch.tanh(z0 / case["cap"])
            z1 = case["cap"] * torch.tanh(z1 / case["cap"])
        z1 = z1.masked_fill(~seen[:, None, :], -math.inf)
        m = torch.maximum(z0.amax(-1, keepdim=True), z1.amax(-1, keepdim=True))
        p0, p1 = torch.exp(z0 - m), torch.exp(z1 - m)
        total = p0.sum(-1, keepdim=True) + p1.sum(-1, keepdim=True)
        o = (p0.view(-1, P) @ vp[h]).view(S, -1, d) + p1 @ vo[:, :, h]
        out[:, h] = torch.where(live, o / total, 0.0)
        lse[:, h] = torch.where(live, m + torch.log(total), -math.inf)[..., 0]
    return out.reshape(S, hq, d), lse.reshape(S, hq)


def _mass_plain(st):
    case, page = st["case"], st["case"]["page"]
    S, hq, d = st["q"].shape
    hkv, L = case["hkv"], st["longest"]
    seen = torch.arange(L, device="cuda") < st["lens"].long()[:, None]
    t = torch.where(seen, torch.arange(L, device="cuda"), 0)
    pages = st["table"].long().gather(1, t // page).clamp(min=0)
    k = st["k_cache"][pages, t % page].float() * SCALES[case["cache"]][0]      # (S, L, hkv, d)
    z = (st["q"].view(S, hkv, -1, d) * (1.0 / math.sqrt(d))) @ k.permute(0, 2, 3, 1)
    if case["cap"]:
        z = case["cap"] * torch.tanh(z / case["cap"])
    p = torch.exp(z - st["lse"].view(S, hkv, -1, 1)).sum(2)
    st["mass_out"].copy_(torch.where(seen[:, None], st["mass"] + p, st["mass_out"]))
    return st["mass_out"]


def _evict_plain(st):
    case, lens = st["case"], st["lens"].long()
    S, hkv, L = st["mass"].shape
    keep, page = case["keep"], case["page"]
    slot = torch.arange(L, device="cuda")
    live = (slot < lens[:, None])[:, None].expand(S, hkv, L)
    newest = torch.where(live, st["held"], -1).amax(-1, keepdim=True)
    safe = live & (st["held"] > newest - case["recent"])
    # safe slots first, then by mass; stable, so equals stay in the order of their slots
    key = torch.where(safe, math.inf, torch.where(live, st["mass"], -1.0))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, slot.expand_as(order))
    kept = live & (rank < keep)
    src = kept & (slot >= keep)
    gone = live & ~kept & (slot < keep)
    n = src.sum(-1)
    nth = torch.arange(L, device="cuda")
    a = torch.where(src, slot, L).sort(-1).values                              # survivors that move
    b = torch.where(gone, slot, L).sort(-1).values                             # and where to
    s, h, i = torch.nonzero(nth < n[..., None], as_tuple=True)
    a, b = a[s, h, i], b[s, h, i]
    first = min(keep, L)
    new = torch.arange(first, device="cuda") < lens[:, None, None]
    for x, y in ((st["mass"], st["mass_out"]), (st["held"], st["held_out"])):
        moved = x[..., :first].clone()
        moved[s, h, b] = x[s, h, a]
        y[..., :first] = torch.where(new, moved, y[..., :first])
    pa, pb = st["table"][s, a // page].long(), st["table"][s, b // page].long()
    for c in (st["k_cache"], st["v_cache"]):
        c = c.view(torch.uint8) if case["cache"] == "e4m3" else c
        c[pb, b % page, h] = c[pa, a % page, h]
    st["lens_out"].copy_(lens.clamp(max=keep))
    return st["k_cache"], st["v_cache"], st["mass_out"], st["held_out"], st["lens_out"]


def run(st):
    case = st["case"]
    if not own:
        return {"append": _append_plain, "prefix": _prefix_plain, "mass": _mass_plain,
                "evict": _evict_plain}[case["op"]](st)
    K = st["K"]
    ks, vs = SCALES[case["cache"]]
    if case["op"] == "append":
        more = dict(slots=st["slots"], mass=st["mass"], held=st["held"]) if case["ledger"] else {}
        q = K.rope_append(st["q"], st["k"], st["v"], st["k_cache"], st["v_cache"], st["table"],
                          st["positions"], st["inv_freq"], seq_ids=st["seq_ids"],
                          interleaved=case["pairs"] == "adjacent", k_scale=ks, v_scale=vs,
                          q_norm=st["wq"], k_norm=st["wk"], eps=EPS, gemma_style=case["gemma"],
                          **more)
        if not case["ledger"]:
            return q, st["k_cache"], st["v_cache"]
        return q, st["k_cache"], st["v_cache"], st["mass"], st["held"]
    if case["op"] == "prefix":
        return K.prefix_attention(st["q"], st["k_cache"], st["v_cache"], st["table"], st["lens"],
                                  st["prefix_pages"], softcap=case["cap"], k_scale=ks, v_scale=vs,
                                  max_len=st["longest"], return_lse=True, ws=st["ws"])
    if case["op"] == "mass":
        return K.attention_mass(st["q"], st["k_cache"], st["table"], st["lens"], st["lse"],
                                st["mass"], softcap=case["cap"], k_scale=ks, max_len=st["longest"],
                                out=st["mass_out"])
    lens = K.cache_evict(st["k_cache"], st["v_cache"], st["table"], st["lens"], st["mass"],
                         st["held"], case["keep"], case["recent"], mass_out=st["mass_out"],
                         held_out=st["held_out"], lens_out=st["lens_out"])
    return st["k_cache"], st["v_cache"], st["mass_out"], st["held_out"], lens


# ------------------------------------------------------------------- 64 bits

def exact(case, seed):
    """The operators' definitions in 64 bits, sequence by sequence."""
    st = prepare(case, seed)
    hkv, d, page = case["hkv"], case["d"], case["page"]
    ks, vs = SCALES[case["cache"]]
    if case["op"] == "append":
        rot = case["rot"]
        i = torch.arange(rot // 2, device="cuda")
        first, second = (i, i + rot // 2) if case["pairs"] == "half" else (2 * i, 2 * i + 1)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                           torch.outer(st["positions"].double(), st["inv_freq"]))[:, None]
        out = []
        for x, w in ((st["q"], st["wq"]), (st["k"], st["wk"])):
            x = x.double()
            norm = torch.linalg.vector_norm(x, dim=-1, keepdim=True).square() / d + EPS
            x = x * norm.rsqrt() * (w.double() + (1.0 if case["gemma"] else 0.0))
            z = torch.complex(x[..., first], x[..., second]) * turn
            x[..., first], x[..., second] = z.real, z.imag
            out.append(x)
        seq, slot = _spread(case)
        where = [(int(c), p % page) for c, p in zip(
            st["table"].cpu()[torch.tensor(seq), torch.tensor(slot) // page], slot)]
        p0, p1 = (torch.tensor(c, device="cuda") for c in zip(*where))
        kc, vc = st["k_cache"].double(), st["v_cache"].double()
        most = 448.0 if case["cache"] == "e4m3" else math.inf
        kc[p0, p1] = (out[1] / ks).clamp(-most, most)
        vc[p0, p1] = (st["v"].double() / vs).clamp(-most, most)
        if not case["ledger"]:
            return out[0], kc, vc
        mass, held = st["mass"].double(), st["held"].clone()
        for t, (s, p) in enumerate(zip(seq, slot)):
            mass[s, :, p], held[s, :, p] = 0.0, st["positions"][t]
        return out[0], kc, vc, mass, held
    lens = _lens(case)
    if case["op"] == "evict":
        kc, vc = st["k_cache"].clone(), st["v_cache"].clone()
        if case["cache"] == "e4m3":
            kc, vc = kc.view(torch.uint8), vc.view(torch.uint8)
        table = st["table"].cpu().numpy()
        mass, held = st["mass"].cpu().numpy(), st["held"].cpu().numpy()
        mass_out, held_out = st["mass_out"].double().cpu(), st["held_out"].cpu()
        for s, n in enumerate(lens):
            moves = []
            for h in range(hkv):
                m, t = mass[s, h, :n], held[s, h, :n]
                safe = t > t.max() - case["recent"] if n else t > 0
                # the last key of lexsort counts first; it is stable
                order = torch.from_numpy(np.lexsort((-m, ~safe)))
                kept = torch.zeros(n, dtype=torch.bool)
                kept[order[:case["keep"]]] = True
                at = torch.arange(n)
                b = at[:case["keep"]][~kept[:case["keep"]]]
                a = at[case["keep"]:][kept[case["keep"]:]]
                where = at[:case["keep"]].clone()
                where[b] = a
                mass_out[s, h, :len(where)] = torch.from_numpy(m)[where].double()
                held_out[s, h, :len(where)] = torch.from_numpy(t)[where]
                moves += [(table[s, i // page], i % page, table[s, j // page], j % page, h)
                          for i, j in zip(a.tolist(), b.tolist())]
            if moves:
                pa, sa, pb, sb, hh = (torch.tensor([int(x) for x in c], device="cuda")
                                      for c in zip(*moves))
                kc[pb, sb, hh], vc[pb, sb, hh] = kc[pa, sa, hh], vc[pa, sa, hh]
        if case["cache"] == "e4m3":
            kc, vc = kc.view(torch.float8_e4m3fn), vc.view(torch.float8_e4m3fn)
        return (kc.double(), vc.double(), mass_out, held_out,
                torch.tensor([min(n, case["keep"]) for n in lens], dtype=torch.int32))
    S, hq, _ = st["q"].shape
    group = hq // hkv
    o = torch.zeros((S, hq, d), dtype=torch.float64, device="cuda")
    lse = torch.full((S, hq), -math.inf, dtype=torch.float64, device="cuda")
    mass = st["mass_out"].double() if case["op"] == "mass" else None
    shared = {}
    if case["op"] == "prefix":                     # read once, for speed only
        pages = st["prefix_pages"].long()
        shared = {h: [(c[pages, :, h].double() * x).flatten(0, 1)
                      for c, x in ((st["k_cache"], ks), (st["v_cache"], vs))] for h in range(hkv)}
    P = case.get("prefix", 0)
    for s, n in enumerate(lens):
        if n == 0:
            continue
        t = torch.arange(P, n, device="cuda")
        pages = st["table"][s][t // page].long()
        for h in range(hkv):
            rows = slice(h * group, (h + 1) * group)
            k = st["k_cache"][pages, t % page, h].double() * ks
            if P:
                k = torch.cat([shared[h][0], k])
            z = torch.einsum("gd,td->gt", st["q"][s, rows].double(), k) / math.sqrt(d)
            if case["cap"]:
                z = case["cap"] * torch.tanh(z / case["cap"])
            if mass is not None:
                p = torch.exp(z - st["lse"][s, rows].double()[:, None])
                mass[s, h, :n] = st["mass"][s, h, :n].double() + p.sum(0)
                continue
            v = torch.cat([shared[h][1], st["v_cache"][pages, t % page, h].double() * vs])
            o[s, rows] = torch.softmax(z, -1) @ v
            lse[s, rows] = torch.logsumexp(z, -1)
    return mass if mass is not None else (o, lse)

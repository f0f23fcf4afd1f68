"""Decode-step operators around the MoE layer, as they are measured.

* ``append``     rotary positions of q and k and the append of k, v to a paged cache
* ``attention``  one new token per sequence over the paged cache
* ``linear``     matrix-vector products with Q4_0 / Q8_0 block weights for a few tokens

Activations are f32, caches fp16, bf16 or e4m3 (with one scale each for keys and values).
``own`` selects the framework's kernels; otherwise ``run`` is the plain torch form.
"""
import math
import random

import torch

own = False

CACHE = {"f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
BLOCK_BYTES = {"q4_0": 18, "q8_0": 34}
GGML_TYPE = {"q4_0": 2, "q8_0": 8}
SCALES = {"f16": (1.0, 1.0), "bf16": (1.0, 1.0), "e4m3": (0.03125, 0.0234375)}   # of keys, of values


def listed():
    return [
        # a single user's token entering the cache: latency only
        dict(name="append one token", op="append", tokens=1, seqs=1, hi=1000, hq=32, hkv=8, d=128,
             rot=128, pairs="half", cache="f16", page=16, layout="nhd"),
        # one decode step of a serving batch, 8-bit cache, adjacent pairs, far positions
        dict(name="append decode batch", op="append", tokens=64, seqs=64, hi=131072, hq=16, hkv=16,
             d=64, rot=64, pairs="adjacent", cache="e4m3", page=64, layout="nhd"),
        # prompts of five sequences entering together, a quarter of each head rotated
        dict(name="append prompts", op="append", tokens=8191, seqs=5, hi=4096, hq=32, hkv=8, d=128,
             rot=32, pairs="half", cache="bf16", page=16, layout="hnd"),
        # the start of a chat
        dict(name="attend one short", op="attention", seqs=1, lo=37, hi=37, hq=32, hkv=8, d=128,
             cache="f16", page=16, layout="nhd", window=0, cap=0.0),
        # a single user with a long context: only the split over the length fills the GPU
        dict(name="attend one long", op="attention", seqs=1, lo=131071, hi=131071, hq=32, hkv=8,
             d=128, cache="f16", page=16, layout="nhd", window=0, cap=0.0),
        # wide heads with a sliding window and capped scores
        dict(name="attend window", op="attention", seqs=32, lo=300, hi=8192, hq=16, hkv=4, d=256,
             cache="bf16", page=32, layout="nhd", window=1024, cap=50.0),
        # a serving batch of ragged lengths, empty rows among them, 8-bit cache
        dict(name="attend batch 8-bit", op="attention", seqs=256, lo=0, hi=2048, hq=32, hkv=8,
             d=128, cache="e4m3", page=64, layout="hnd", window=0, cap=0.0),
        # a head of its own for each query head, pages that end inside any tile
        dict(name="attend every head", op="attention", seqs=48, lo=1, hi=2500, hq=16, hkv=16, d=64,
             cache="f16", page=24, layout="nhd", window=0, cap=0.0),
        # the joint q, k, v projection of one token at the decode layer's width
        dict(name="linear one token", op="linear", tokens=1, n=6144, k=2816, quant="q4_0",
             residual=False),
        # an output head over a large vocabulary for one token
        dict(name="linear vocabulary", op="linear", tokens=1, n=262144, k=2816, quant="q4_0",
             residual=False),
        # attention output projection of a decode batch, added to the residual stream
        dict(name="linear batch", op="linear", tokens=16, n=4096, k=8192, quant="q4_0",
             residual=True),
        # odd sizes: rows that fill no tile, a last half tile of columns, 8-bit weights
        dict(name="linear odd", op="linear", tokens=5, n=5003, k=1056, quant="q8_0",
             residual=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "linear"])
    if op == "linear":
        quant = rng.choice(["q4_0", "q4_0", "q8_0"])
        k = 32 * _log(rng, 8, 256)
        most = 1 << 29 if quant == "q4_0" else 1 << 28
        return dict(op=op, tokens=_log(rng, 1, 16), n=_log(rng, 64, min(262144, most // k)), k=k,
                    quant=quant, residual=rng.random() < 0.5)
    d = rng.choice([64, 80, 96, 128, 128, 192, 256])
    hkv = rng.choice([1, 2, 4, 8, 8, 16])
    hq = hkv * rng.choice([1, 2, 3, 4, 5, 8]) if hkv < 16 else hkv * rng.choice([1, 2])
    cache = rng.choice(["f16", "bf16", "e4m3"])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    layout = rng.choice(["nhd", "hnd"])
    if op == "append":
        tokens = _log(rng, 1, max(2, min(8192, (1 << 26) // ((hq + 2 * hkv) * d))))
        decode = rng.random() < 0.5 and tokens <= 512
        return dict(op=op, tokens=tokens, seqs=tokens if decode else rng.randint(1, min(tokens, 16)),
                    hi=_log(rng, 64, 131072) if decode else max(64, tokens), hq=hq, hkv=hkv, d=d,
                    rot=rng.choice([d, d, d // 2]), pairs=rng.choice(["half", "adjacent"]),
                    cache=cache, page=page, layout=layout)
    keys = (1 << 27) // (hkv * d)                  # of the whole batch, at most
    seqs = _log(rng, 1, 256)
    hi = _log(rng, 16, max(17, min(131072, keys // seqs)))
    return dict(op=op, seqs=seqs, lo=rng.choice([0, 1, hi // 2, hi]), hi=hi, hq=hq, hkv=hkv, d=d,
                cache=cache, page=page, layout=layout,
                window=rng.choice([0, 0, max(1, hi // 3)]), cap=rng.choice([0.0, 0.0, 30.0]))


def _lens(case):
    """Sequence lengths of an attention case: its own, whatever the seed."""
    r = random.Random(case["seqs"] * 1000003 + case["hi"])
    lens = [r.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]
    lens[r.randrange(len(lens))] = case["hi"]
    return lens


def _spread(case):
    """(sequence, position) of every token of an append case."""
    r = random.Random(case["tokens"] * 1000003 + case["hi"])
    T, S = case["tokens"], case["seqs"]
    if S == T:                                     # one new token each
        return list(range(T)), [r.randrange(case["hi"]) for _ in range(T)]
    cuts = sorted(r.sample(range(1, T), S - 1)) if S > 1 else []
    seq, pos = [], []
    for s, (a, b) in enumerate(zip([0] + cuts, cuts + [T])):
        first = r.randrange(max(1, case["hi"] - (b - a)))
        seq += [s] * (b - a)
        pos += range(first, first + b - a)
    return seq, pos


def work(case):
    if case["op"] == "linear":
        T, n, k = case["tokens"], case["n"], case["k"]
        b = n * (k // 32) * BLOCK_BYTES[case["quant"]] + 4 * T * (k + n * (2 if case["residual"] else 1))
        return {"bytes": b, "flops": 2 * T * n * k}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    e = 1 if case["cache"] == "e4m3" else 2
    if case["op"] == "append":
        T = case["tokens"]
        return {"bytes": T * ((2 * hq + 2 * hkv) * d * 4 + 2 * hkv * d * e),
                "flops": T * (hq + hkv) * case["rot"] * 3}
    keys = sum(min(n, case["window"]) if case["window"] else n for n in _lens(case))
    return {"bytes": 2 * keys * hkv * d * e + case["seqs"] * hq * (2 * d + 1) * 4,
            "flops": 4 * keys * hq * d}


# ------------------------------------------------------------------- inputs

def _pages(case, need, g):
    """Caches of a pool with a few pages more than `need` (pages per sequence),
    and the page table; entries behind a sequence's last page are -1."""
    hkv, d, page = case["hkv"], case["d"], case["page"]
    total, width = sum(need) + 3, max(need) + 1
    shape = (total, page, hkv, d) if case["layout"] == "nhd" else (total, hkv, page, d)
    caches = []
    for scale in SCALES[case["cache"]]:
        c = torch.empty(shape, dtype=CACHE[case["cache"]], device="cuda")
        for at in range(0, total, 4096):
            part = torch.randn((min(4096, total - at),) + shape[1:], generator=g, device="cuda")
            c[at:at + 4096].copy_(part / scale)
        caches.append(c if case["layout"] == "nhd" else c.transpose(1, 2))
    free = torch.randperm(total, generator=g, device="cuda", dtype=torch.int32)
    counts = torch.tensor(need, device="cuda")
    first = torch.cumsum(counts, 0) - counts
    col = torch.arange(width, device="cuda")
    at = (first[:, None] + col).clamp(max=total - 1)
    table = torch.where(col < counts[:, None], free[at], -1).to(torch.int32)
    return caches, table.contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    st = {"case": case}
    if own:
        from linuxnightmaresuite_b200 import kernels
        st["K"] = kernels
    if case["op"] == "linear":
        n, k, T = case["n"], case["k"], case["tokens"]
        nb, size = n * (k // 32), BLOCK_BYTES[case["quant"]]
        raw = torch.empty((nb, size), dtype=torch.uint8, device="cuda")
        for at in range(0, nb, 1 << 22):
            m = min(1 << 22, nb - at)
            raw[at:at + m, 2:] = torch.randint(0, 256, (m, size - 2), generator=g, device="cuda",
                                               dtype=torch.uint8)
            d = torch.randn((m, 1), generator=g, device="cuda").mul_(0.3).exp_().mul_(
                0.006 if size == 18 else 0.0004)
            raw[at:at + m, :2] = d.half().view(torch.uint8)
        st["x"] = torch.randn((T, k), generator=g, device="cuda")
        st["residual"] = torch.randn((T, n), generator=g, device="cuda") if case["residual"] else None
        st["raw"] = raw.view(n, -1)
        if own:                                    # laid out once, at load time
            st["w"] = kernels.LinearWeights(st["raw"], GGML_TYPE[case["quant"]], n, k)
        return st
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    if case["op"] == "append":
        seq, pos = _spread(case)
        last = [0] * case["seqs"]
        for s, p in zip(seq, pos):
            last[s] = max(last[s], p)
        # only the pages that are written exist; positions before them share the pool's first page
        (st["k_cache"], st["v_cache"]), table = _pages(
            case, [min(p // page + 1, -(-case["tokens"] // page) + 2) for p in last], g)
        cols = torch.arange(max(p // page for p in last) + 1, device="cuda")
        lastcol = torch.tensor([p // page for p in last], device="cuda")[:, None]
        held = torch.tensor([min(p // page + 1, -(-case["tokens"] // page) + 2) for p in last],
                            device="cuda")[:, None]
        at = cols - (lastcol + 1 - held)
        st["table"] = torch.where((at >= 0) & (at < held), table.gather(1, at.clamp(
            0, table.shape[1] - 1)), -1).to(torch.int32).contiguous()
        st["positions"] = torch.tensor(pos, dtype=torch.int32, device="cuda")
        st["seq_ids"] = None if case["seqs"] == case["tokens"] else torch.tensor(
            seq, dtype=torch.int32, device="cuda")
        i = torch.arange(case["rot"] // 2, dtype=torch.float64, device="cuda")
        st["inv_freq"] = 10000.0 ** (-2.0 * i / case["rot"])
        # as the joint projection leaves them: q, k, v of a token side by side
        qkv = torch.randn((case["tokens"], (hq + 2 * hkv) * d), generator=g, device="cuda")
        st["q"] = qkv[:, :hq * d].unflatten(1, (hq, d))
        st["k"] = qkv[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
        st["v"] = qkv[:, (hq + hkv) * d:].unflatten(1, (hkv, d))
        return st
    lens = _lens(case)
    (st["k_cache"], st["v_cache"]), st["table"] = _pages(case, [-(-n // page) for n in lens], g)
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    st["longest"] = max(lens)
    st["q"] = 1.5 * torch.randn((case["seqs"], hq, d), generator=g, device="cuda")
    if own:
        st["ws"] = kernels.paged_attention_workspace(case["seqs"], hq, hkv, d, "cuda")
    return st


# ------------------------------------------------------------------- one pass

def _append_plain(st):
    case, q, k, v = st["case"], st["q"], st["k"], st["v"]
    h = case["rot"] // 2
    angle = st["positions"].double()[:, None, None] * st["inv_freq"]
    cos, sin = angle.cos().float(), angle.sin().float()

    def turn(x):
        r, rest = x[..., :2 * h], x[..., 2 * h:]
        if case["pairs"] == "half":
            a, b = r[..., :h], r[..., h:]
            return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
        a, b = r[..., 0::2], r[..., 1::2]
        return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)

    pos = st["positions"].long()
    rows = st["seq_ids"].long() if st["seq_ids"] is not None else torch.arange(len(pos), device="cuda")
    page = st["table"][rows, pos // case["page"]].long()
    slot = pos % case["page"]
    for x, c, scale in ((turn(k), st["k_cache"], SCALES[case["cache"]][0]),
                        (v, st["v_cache"], SCALES[case["cache"]][1])):
        if case["cache"] == "e4m3":
            c.view(torch.uint8)[page, slot] = (x / scale).clamp(-448, 448).to(c.dtype).view(torch.uint8)
        else:
            c[page, slot] = x.to(c.dtype)
    return turn(q), st["k_cache"], st["v_cache"]


def _attention_plain(st):
    case, q = st["case"], st["q"]
    S, hq, d = q.shape
    hkv, page, window = case["hkv"], case["page"], case["window"]
    L = min(window, st["longest"]) if window else st["longest"]
    lens = st["lens"].long()[:, None]
    t = torch.arange(L, device="cuda") + ((lens - L).clamp(min=0) if window else 0 * lens)
    seen = t < lens
    t = torch.where(seen, t, 0)
    pages = st["table"].long().gather(1, t // page).clamp(min=0)
    ks, vs = SCALES[case["cache"]]
    k = st["k_cache"][pages, t % page].float() * ks            # (S, L, hkv, d)
    v = st["v_cache"][pages, t % page].float() * vs
    qg = q.view(S, hkv, hq // hkv, d) * (1.0 / math.sqrt(d))
    s = qg @ k.permute(0, 2, 3, 1)                             # (S, hkv, group, L)
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    s = s.masked_fill(~seen[:, None, None, :], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    o = (p @ v.permute(0, 2, 1, 3)) / torch.where(total == 0, 1.0, total)
    return o.reshape(S, hq, d), (m + torch.log(total)).reshape(S, hq)


def _linear_plain(st):
    case = st["case"]
    size = BLOCK_BYTES[case["quant"]]
    blocks = st["raw"].view(-1, size)
    d = blocks[:, :2].contiguous().view(torch.float16).float()
    q = blocks[:, 2:]
    if size == 18:
        q = torch.cat([q & 15, q >> 4], 1).float() - 8.0
    else:
        q = q.contiguous().view(torch.int8).float()
    y = st["x"] @ (d * q).view(case["n"], case["k"]).t()
    return y if st["residual"] is None else y + st["residual"]


def run(st):
    case = st["case"]
    if not own:
        return {"append": _append_plain, "attention": _attention_plain,
                "linear": _linear_plain}[case["op"]](st)
    K = st["K"]
    if case["op"] == "linear":
        return K.linear(st["x"], st["w"], residual=st["residual"])
    ks, vs = SCALES[case["cache"]]
    if case["op"] == "append":
        q = K.rope_append(st["q"], st["k"], st["v"], st["k_cache"], st["v_cache"], st["table"],
                          st["positions"], st["inv_freq"], seq_ids=st["seq_ids"],
                          interleaved=case["pairs"] == "adjacent", k_scale=ks, v_scale=vs)
        return q, st["k_cache"], st["v_cache"]
    return K.paged_attention(st["q"], st["k_cache"], st["v_cache"], st["table"], st["lens"],
                             window=case["window"], softcap=case["cap"], k_scale=ks, v_scale=vs,
                             max_len=st["longest"], return_lse=True, ws=st["ws"])


# ------------------------------------------------------------------- 64 bits

def exact(case, seed):
    """The operators' definitions in 64 bits, sequence by sequence or a few rows at a time."""
    st = prepare(case, seed)
    if case["op"] == "linear":
        n, k = case["n"], case["k"]
        size = BLOCK_BYTES[case["quant"]]
        x = st["x"].double()
        y = torch.empty((case["tokens"], n), dtype=torch.float64, device="cuda")
        for a in range(0, n, 8192):
            b = st["raw"][a:a + 8192].reshape(-1, k // 32, size)
            w = torch.empty(b.shape[:2] + (32,), dtype=torch.float64, device="cuda")
            if size == 18:
                w[..., :16] = (b[..., 2:] % 16).double() - 8
                w[..., 16:] = (b[..., 2:] // 16).double() - 8
            else:
                u = b[..., 2:].double()
                w.copy_(torch.where(u > 127, u - 256, u))
            w *= b[..., :2].contiguous().view(torch.float16).double()
            y[:, a:a + 8192] = torch.einsum("tk,nk->tn", x, w.flatten(1))
        return y if st["residual"] is None else y + st["residual"].double()
    ks, vs = SCALES[case["cache"]]
    page = case["page"]
    if case["op"] == "append":
        rot = case["rot"]
        i = torch.arange(rot // 2, device="cuda")
        first, second = (i, i + rot // 2) if case["pairs"] == "half" else (2 * i, 2 * i + 1)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                           torch.outer(st["positions"].double(), st["inv_freq"]))[:, None]
        out = []
        for x in (st["q"].double(), st["k"].double()):
            z = torch.complex(x[..., first], x[..., second]) * turn
            x[..., first], x[..., second] = z.real, z.imag
            out.append(x)
        seq, pos = _spread(case)
        where = [(int(c), p % page) for c, p in zip(
            st["table"].cpu()[torch.tensor(seq), torch.tensor(pos) // page], pos)]
        p0, p1 = (torch.tensor(c, device="cuda") for c in zip(*where))
        kc, vc = st["k_cache"].double(), st["v_cache"].double()
        most = 448.0 if case["cache"] == "e4m3" else math.inf
        kc[p0, p1] = (out[1] / ks).clamp(-most, most)
        vc[p0, p1] = (st["v"].double() / vs).clamp(-most, most)
        return out[0], kc, vc
    S, hq, d = st["q"].shape
    hkv = case["hkv"]
    o = torch.zeros((S, hq, d), dtype=torch.float64, device="cuda")
    lse = torch.full((S, hq), -math.inf, dtype=torch.float64, device="cuda")
    for s, n in enumerate(_lens(case)):
        a = max(0, n - case["window"]) if case["window"] else 0
        if n == a:
            continue
        t = torch.arange(a, n, device="cuda")
        pages = st["table"][s][t // page].long()
        for h in range(hkv):
            k = st["k_cache"][pages, t % page, h].double() * ks
            v = st["v_cache"][pages, t % page, h].double() * vs
            rows = slice(h * hq // hkv, (h + 1) * hq // hkv)
            z = torch.einsum("gd,td->gt", st["q"][s, rows].double(), k) / math.sqrt(d)
            if case["cap"]:
                z = case["cap"] * torch.tanh(z / case["cap"])
            o[s, rows] = torch.softmax(z, -1) @ v
            lse[s, rows] = torch.logsumexp(z, -1)
    return o, lse

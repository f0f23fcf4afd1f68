"""Norms of q and k with the append, attention weight per slot, eviction by it:
each against a plain 64-bit form, at the sizes and masks where it can go wrong."""
import math

import pytest
import torch

from linuxnightmaresuite_b200 import kernels as K

from ._attention import BF16, E4M3, F16, SCALES, Cache, check_stored, rotate
from .test_gpu_attention import randn

pytestmark = pytest.mark.gpu


def i32(*v):
    return torch.tensor(v, dtype=torch.int32).cuda()


# --------------------------------------------------------------------------- append with norms

def normed(x, w, eps, gemma):
    """x (T, H, d) f64 and the bound of an f32 form: a sum of up to 256 squares in
    parts of 8 and a tree (20 roundings of 2^-24), its root and quotient (half of that and
    three more), the weight and two products (three): 2^-19 of the value in all."""
    if w is None:
        return x, torch.zeros_like(x)
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * (w.double() + (1.0 if gemma else 0.0))
    return y, y.abs() * 2.0 ** -19


def turned(x, bound, positions, freq, interleaved):
    """A pair's errors turn with it: |cos| e0 + |sin| e1 <= e0 + e1 for both."""
    y, b = rotate(x, positions, freq, interleaved)
    rot = 2 * freq.numel()
    i = torch.arange(rot // 2, device=x.device)
    e0, e1 = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    total = bound.clone()
    total[..., e0] = total[..., e1] = (bound[..., e0] + bound[..., e1])
    return y, total * (1 + 2.0 ** -20) + b


@pytest.mark.parametrize("dtype", [F16, BF16, E4M3])
@pytest.mark.parametrize("hq,hkv,d,rot,interleaved,page,gemma,gap", [
    (8, 2, 128, 128, False, 16, False, 4),
    (16, 8, 128, 64, False, 16, True, 0),      # several rows for each group of lanes
    (4, 4, 64, 32, True, 5, False, 4),
    (3, 1, 80, 80, False, 1, True, 4),
    (5, 5, 256, 64, False, 64, False, 4),
    (4, 2, 256, 256, True, 8, True, 0),
    (2, 1, 16, 6, False, 7, False, 4),         # three pairs: elements one by one
    (1, 1, 16, 14, True, 3, True, 4),
    (3, 2, 96, 96, False, 4, False, 1),        # rows off 16 bytes
    (6, 3, 96, 0, False, 8, False, 4),         # nothing turns
    (0, 2, 64, 64, False, 4, False, 0),        # keys alone
])
def test_norm_append(dtype, hq, hkv, d, rot, interleaved, page, gemma, gap):
    lens = [page * 3 + 2, 1, 2 * page]
    c = Cache(lens, page, hkv, d, dtype, "hnd" if d == 96 else "nhd", seed=d)
    before = (c.k.clone().view(torch.uint8), c.v.clone().view(torch.uint8))
    seq = [0, 0, 0, 2, 1, 2, 0]
    at = [lens[0] - 1, 0, page, 2 * page - 1, 0, page - 1, 2 * page]
    pos = [70000 + 13 * i for i in range(7)]
    qkv = 3.0 * randn(len(seq), (hq + 2 * hkv) * d + gap, seed=rot)
    q = qkv[:, :hq * d].unflatten(1, (hq, d)) if hq else None
    k = qkv[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
    v = qkv[:, (hq + hkv) * d:(hq + 2 * hkv) * d].unflatten(1, (hkv, d))
    freq = K.rope_inv_freq(rot) if rot else None
    wq, wk = (0.3 * randn(d, seed=s) + (0.0 if gemma else 1.0) for s in (1, 2))
    width = c.table.shape[1] * page
    mass, held = randn(3, hkv, width, seed=9), torch.full((3, hkv, width), -5, dtype=torch.int32,
                                                          device="cuda")
    want_mass, want_held = mass.clone(), held.clone()
    status = i32(0)
    out = K.rope_append(q, k, v, *c.args, i32(*pos), freq, i32(*seq), interleaved, status=status,
                        q_norm=wq, k_norm=wk, eps=1e-5, gemma_style=gemma, slots=i32(*at),
                        mass=mass, held=held, **c.scales)
    f = freq if rot else torch.zeros(0, dtype=torch.float64, device="cuda")
    if hq:
        yq, bq = turned(*normed(q.double(), wq, 1e-5, gemma), i32(*pos), f, interleaved)
        assert ((out.double() - yq).abs() <= bq).all()
    yk, bk = turned(*normed(k.double(), wk, 1e-5, gemma), i32(*pos), f, interleaved)
    touched = torch.zeros(c.k.shape[:2], dtype=torch.bool, device="cuda")
    for i, (s, a) in enumerate(zip(seq, at)):
        pages, slots = c.where(s, [a])
        touched[pages, slots] = True
        ks, vs = SCALES[dtype]
        check_stored(c.k[pages, slots][0], yk[i], bk[i], dtype, ks)
        check_stored(c.v[pages, slots][0], v[i].double(), 0 * bk[i], dtype, vs)
        want_mass[s, :, a], want_held[s, :, a] = 0.0, pos[i]
    for new, old in zip((c.k, c.v), before):
        assert torch.equal(new.view(torch.uint8)[~touched], old[~touched])
    assert torch.equal(mass, want_mass) and torch.equal(held, want_held)
    assert status.item() == 0


def test_norm_append_parts_alone():
    """Norms of q or k alone; slots without norms gives what the plain append at those
    slots gives, bit by bit."""
    hq, hkv, d, page = 4, 2, 128, 4
    c = Cache([8, 8], page, hkv, d, F16)
    q, k, v = randn(2, hq, d), randn(2, hkv, d, seed=1), randn(2, hkv, d, seed=2)
    freq, w = K.rope_inv_freq(d), 1.0 + 0.1 * randn(d, seed=3)
    pos, at = i32(100, 2000), i32(5, 2)
    for wq, wk in ((w, None), (None, w)):
        out = K.rope_append(q, k, v, *c.args, pos, freq, q_norm=wq, k_norm=wk, slots=at)
        y, b = turned(*normed(q.double(), wq, 1e-6, False), pos, freq, False)
        assert ((out.double() - y).abs() <= b).all()
        y, b = turned(*normed(k.double(), wk, 1e-6, False), pos, freq, False)
        for s, a in ((0, 5), (1, 2)):
            check_stored(c.k[c.where(s, [a])][0], y[s], b[s], F16, 1.0)
    # the plain form at the positions, the other at slots that are the positions
    plain = K.rope_append(q, k, v, *c.args, at, freq)
    kk, vv = c.k.clone(), c.v.clone()
    c.k[c.where(0, [5])], c.v[c.where(1, [2])] = 0.0, 0.0
    assert torch.equal(K.rope_append(q, k, v, *c.args, at, freq, slots=at), plain)
    assert torch.equal(c.k.view(torch.int16), kk.view(torch.int16))
    assert torch.equal(c.v.view(torch.int16), vv.view(torch.int16))


def test_norm_append_skips_and_reports():
    hkv, d, page = 2, 64, 4
    c = Cache([8] * 5, page, hkv, d, BF16)
    old_k = c.k.clone()
    table = c.table_d.clone()
    table[2, 1] = c.k.shape[0]
    q, k, v = randn(6, 4, d), randn(6, hkv, d, seed=1), randn(6, hkv, d, seed=2)
    out = torch.full_like(q, 7.0)
    w, freq, status = torch.ones(d, device="cuda"), K.rope_inv_freq(d), i32(0)
    mass = torch.full((5, hkv, 7), 3.0, device="cuda")
    held = torch.full((5, hkv, 7), 3, dtype=torch.int32, device="cuda")
    #         padding, padding, bad page, behind the ledger, no such sequence, fine
    pos, at, seq = i32(-1, 4, 9, 9, 9, 9), i32(0, -1, 6, 7, 0, 5), i32(0, 1, 2, 3, 5, 4)
    K.rope_append(q, k, v, c.k, c.v, table, pos, freq, seq, q_out=out, status=status, q_norm=w,
                  k_norm=w, slots=at, mass=mass, held=held)
    assert status.item() == K.STATUS_BAD_PAGE
    assert (out[:2] == 7.0).all() and not (out[2:] == 7.0).any()
    changed = torch.zeros(c.k.shape[:2], dtype=torch.bool, device="cuda")
    changed[c.where(4, [5])] = True
    assert torch.equal(c.k[~changed].view(torch.int16), old_k[~changed].view(torch.int16))
    assert not torch.isnan(c.k[changed]).any()
    want = torch.full_like(mass, 3.0)
    want[4, :, 5] = 0.0
    assert torch.equal(mass, want) and (held[4, :, 5] == 9).all() and (held == 3).sum() == 5 * hkv * 7 - hkv
    status.zero_()
    # a row of zeros: eps alone is under the root
    z = torch.zeros_like(k)
    K.rope_append(q, z, v, *c.args, i32(0, 1, 2, 3, 4, -1), freq, seq, q_norm=w, k_norm=w)
    assert (c.k[c.where(0, [0])] == 0).all()


# --------------------------------------------------------------------------- mass

def weights(q, kd, lse, scale, window=0, cap=0.0):
    """(weight per key head and key, its bound), 64 bits: q (hq, d), kd (n, hkv, d).
    A score is off by ds = 2^-18 of its products' magnitudes as in the attention (a cap adds
    2^-21 cap); the exponent s - lse by that and a rounding of 2^-23 of |s| + |lse|
    each for factor, product and difference; exp2 by 2^-22; heads and mass add 2^-24 each."""
    hq, hkv = q.shape[0], kd.shape[1]
    kr = kd.repeat_interleave(hq // hkv, 1)
    s = torch.einsum("hd,nhd->hn", q, kr) * scale
    S = torch.einsum("hd,nhd->hn", q.abs(), kr.abs()) * abs(scale)
    if cap:
        s = cap * torch.tanh(s / cap)
    p = torch.exp(s - lse[:, None])
    n = kd.shape[0]
    if window and n > window:
        p[:, :n - window] = 0
    tol = p * (S * 2.0 ** -18 + cap * 2.0 ** -21 + (s.abs() + lse[:, None].abs()) * 2.0 ** -21
               + 2.0 ** -21 + hq // hkv * 2.0 ** -24) * 1.01
    return (x.view(hkv, hq // hkv, n).sum(1) for x in (p, tol))


def lse_of(c, q, scale, window=0, cap=0.0):
    return K.paged_attention(q, *c.args, c.lens, scale, window, cap, return_lse=True, **c.scales)[1]


def check_mass(c, q, lse, mass, out, scale, window=0, cap=0.0):
    for s, kd in enumerate(c.kd):
        n = kd.shape[0]
        if n:
            p, tol = weights(q[s].double(), kd, lse[s].double(), scale, window, cap)
            want = mass[s, :, :n].double() + p
            err = (out[s, :, :n].double() - want).abs()
            assert (err <= tol + want.abs() * 2.0 ** -23).all(), (s, err.max().item())
        assert torch.equal(out[s, :, n:], mass[s, :, n:])


@pytest.mark.parametrize("dtype", [F16, BF16, E4M3])
@pytest.mark.parametrize("lens,page,hq,hkv,d,layout", [
    ([1, 0, 37], 16, 8, 2, 128, "nhd"),
    ([300, 31, 32, 33], 7, 3, 1, 64, "hnd"),
    ([65, 600], 1, 16, 2, 256, "nhd"),          # a group of 8 heads, one slot a page
    ([129], 64, 20, 2, 80, "nhd"),              # ten heads: two groups
    ([1000, 5], 24, 5, 5, 192, "hnd"),
    ([70, 2], 16, 72, 2, 128, "nhd"),           # 36 heads: the keys are read twice
    ([50, 0, 33], 8, 34, 2, 256, "hnd"),        # 17 heads of 256: of a bf16 cache twice
])
def test_attention_mass(dtype, lens, page, hq, hkv, d, layout):
    c = Cache(lens, page, hkv, d, dtype, layout, seed=hq)
    q, scale = randn(len(lens), hq, d, seed=3), d ** -0.5
    lse = lse_of(c, q, scale)
    mass = randn(len(lens), hkv, max(lens) + 3, seed=4).abs()
    status = i32(0)
    out = K.attention_mass(q, c.k, c.table_d, c.lens, lse, mass, k_scale=c.k_scale,
                           out=mass.clone(), status=status)
    check_mass(c, q, lse, mass, out, scale)
    again = mass.clone()                            # in place, launched for another length
    assert K.attention_mass(q, c.k, c.table_d, c.lens, lse, again, k_scale=c.k_scale, max_len=9,
                            status=status) is again
    assert torch.equal(again, out)
    assert status.item() == 0
    for s, n in enumerate(lens):                    # the weights of a head add up to one
        if n:
            got = (out - mass)[s].double().sum(-1)
            assert (got - hq // hkv).abs().max() < (hq // hkv) * 1e-4


@pytest.mark.parametrize("dtype", [F16, BF16, E4M3])
def test_attention_mass_window_cap_strides(dtype):
    lens, d = [500, 40, 0, 77], 96
    c = Cache(lens, 8, 2, d, dtype, seed=1)
    wide = randn(4, 8 * d + 8, seed=2)              # rows of q that stride
    q = wide[:, :8 * d].unflatten(1, (8, d))
    for window, cap, scale in ((64, 0.0, 0.2), (0, 5.0, 1.0), (50, 30.0, -0.1), (0, 1e-6, 0.1)):
        lse = lse_of(c, q, scale, window, cap)
        mass = randn(4, 2, 500, seed=4)
        out = K.attention_mass(q, c.k, c.table_d, c.lens, lse, mass, scale, window, cap, c.k_scale,
                               out=mass.clone())
        check_mass(c, q, lse, mass, out, scale, window, cap)


def test_attention_mass_bad_pages_and_rows_of_nothing():
    lens, d = [40, 40, 12], 64
    c = Cache(lens, 8, 2, d, F16, seed=1)
    q = randn(3, 4, d, seed=2)
    lse = lse_of(c, q, d ** -0.5)
    mass = randn(3, 2, 30, seed=3)
    table, status = c.table_d.clone(), i32(0)
    table[0, 1] = -3
    lse[1, 0] = -math.inf                           # a head that has seen nothing
    out = K.attention_mass(q, c.k, table, c.lens, lse, mass, out=mass.clone(), status=status)
    assert status.item() == K.STATUS_BAD_PAGE       # the page, and lengths behind the ledger
    for s in range(3):
        n = min(lens[s], 30)
        p, tol = weights(q[s].double(), c.kd[s][:n], lse[s].double(), d ** -0.5)
        if s == 0:
            p[:, 8:16] = 0
        if s == 1:
            p[0] = weights(q[s, 1:2].double(), c.kd[s][:n, :1], lse[s, 1:2].double(), d ** -0.5).__next__()[0]
            tol = tol.nan_to_num(0, 0, 0) + 1e-5
        want = mass[s, :, :n].double() + p
        assert ((out[s, :, :n] - want).abs() <= tol + want.abs() * 2.0 ** -23).all(), s
    assert torch.equal(out[0, :, 8:16], mass[0, :, 8:16])
    # lengths below zero are empty; a batch without sequences is no error
    K.attention_mass(q, c.k, table, i32(-1, 0, -9), lse, mass, out=out.fill_(5.0))
    assert (out == 5.0).all()
    e = torch.empty(0, 4, d, device="cuda")
    K.attention_mass(e, c.k, table[:0], c.lens[:0], lse[:0], mass[:0])


# --------------------------------------------------------------------------- eviction

def evict_plain(lens, mass, held, keep, recent):
    """[(slots that move, where to)] of each (sequence, head)."""
    moves = {}
    for s, n in enumerate(lens):
        for h in range(mass.shape[1]):
            if n <= keep:
                moves[s, h] = ([], [])
                continue
            m, t = mass[s, h, :n].tolist(), held[s, h, :n].tolist()
            m = [-math.inf if x != x else x + 0.0 for x in m]
            nan = [x != x for x in mass[s, h, :n].tolist()]
            since = max(t) - recent
            order = sorted(range(n), key=lambda i: (t[i] <= since, nan[i], -m[i], i))
            kept = set(order[:keep])
            moves[s, h] = ([i for i in range(keep, n) if i in kept],
                           [i for i in range(keep) if i not in kept])
    return moves


def check_evict(lens, page, hkv, d, dtype, keep, recent, mass, held, layout="nhd", in_place=True,
                max_len=0):
    c = Cache(lens, page, hkv, d, dtype, layout, seed=keep)
    moves = evict_plain(lens, mass.cpu(), held.cpu(), keep, recent)
    bits = torch.uint8 if dtype == E4M3 else torch.int16
    want = [c.k.clone().view(bits), c.v.clone().view(bits)]
    wm, wh = mass.clone(), held.clone()
    for (s, h), (a, b) in moves.items():
        assert len(a) == len(b)
        if a:
            for w in want:
                w[(*c.where(s, b), h)] = w[(*c.where(s, a), h)]
            wm[s, h, b], wh[s, h, b] = wm[s, h, a], wh[s, h, a]
    status = i32(0)
    if in_place:
        mass, held = mass.clone(), held.clone()
        got = K.cache_evict(*c.args, c.lens, mass, held, keep, recent, max_len=max_len, status=status)
        assert got is c.lens
        assert torch.equal(mass.view(torch.int32), wm.view(torch.int32)) and torch.equal(held, wh)
    else:
        mo = torch.full((len(lens), hkv, keep + 2), 9.0, device="cuda")
        ho = torch.full(mo.shape, 9, dtype=torch.int32, device="cuda")
        got = K.cache_evict(*c.args, c.lens, mass, held, keep, recent, mo, ho,
                            torch.empty_like(c.lens), max_len, status)
        for s, n in enumerate(lens):
            n = min(n, keep)
            for x, y in ((mo, wm), (ho, wh)):
                assert torch.equal(x[s, :, :n].view(torch.int32), y[s, :, :n].view(torch.int32))
                assert (x[s, :, n:] == 9).all()
    assert got.tolist() == [min(max(n, 0), keep) for n in lens]
    assert torch.equal(c.k.view(bits), want[0]) and torch.equal(c.v.view(bits), want[1])
    assert status.item() == 0


def ledger(seqs, hkv, width, seed=0, ties=False):
    g = torch.Generator().manual_seed(seed)
    m = torch.randn((seqs, hkv, width), generator=g).exp()
    if ties:
        m = (m * 2).round() / 2
    t = torch.rand((seqs, hkv, width), generator=g).argsort(-1).to(torch.int32) * 2 + 5
    return m.cuda(), t.cuda()


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("dtype", [F16, BF16, E4M3])
@pytest.mark.parametrize("lens,page,hkv,d,keep,recent,layout", [
    ([9, 0, 8, 1], 4, 2, 64, 8, 3, "nhd"),
    ([50, 700, 20], 7, 3, 128, 40, 0, "hnd"),
    ([2, 3], 1, 1, 16, 1, 1, "nhd"),            # the newest token alone
    ([333], 16, 2, 256, 300, 300, "nhd"),       # a window of the last tokens
    ([1000, 1025], 24, 2, 80, 999, 100, "hnd"),
    ([5000], 32, 1, 64, 1234, 77, "nhd"),       # several CTAs
])
def test_evict(dtype, in_place, lens, page, hkv, d, keep, recent, layout):
    m, t = ledger(len(lens), hkv, max(lens) + 3, seed=keep)
    check_evict(lens, page, hkv, d, dtype, keep, recent, m, t, layout, in_place)
    m, t = ledger(len(lens), hkv, max(lens), seed=keep + 1, ties=True)
    check_evict(lens, page, hkv, d, dtype, keep, recent, m, t, layout, in_place, max(lens))


def test_evict_special_masses():
    """Ties of zeros of both signs, infinities, NaN, denormals, all equal."""
    lens, width = [64] * 6, 70
    m, t = ledger(6, 2, width, seed=1)
    m[0] = 0.0
    m[0, :, ::3] = -0.0
    m[1, :, 5:20] = math.nan
    m[2, :, ::4], m[2, :, 1::4] = math.inf, -math.inf
    m[3] = torch.arange(width, device="cuda") * 1e-45
    m[4] = -m[4]
    m[5] = 1.5
    for keep, recent in ((63, 0), (32, 5), (50, 50), (1, 0)):
        check_evict(lens, 8, 2, 64, F16, keep, recent, m, t)


@pytest.mark.parametrize("n,keep", [(40000, 39999), (40000, 128), (30011, 15000)])
def test_evict_long(n, keep):
    m, t = ledger(1, 2, n, seed=n, ties=True)
    check_evict([n], 64, 2, 64, F16, keep, keep // 3, m, t)


def test_evict_reports():
    lens, d = [20, 30, 20], 64
    c = Cache(lens, 4, 2, d, F16)
    m, t = ledger(3, 2, 32)
    before = (c.k.clone().view(torch.int16), m.clone(), t.clone())
    status = i32(0)
    # longer than told: left alone, and reported
    got = K.cache_evict(*c.args, c.lens, m, t, 8, max_len=25, status=status)
    assert status.item() == K.STATUS_BAD_PAGE and got.tolist() == [8, 30, 8]
    assert torch.equal(m[1], before[1][1]) and torch.equal(t[1], before[2][1])
    pages, slots = c.where(1, range(30))
    assert torch.equal(c.k[pages, slots].view(torch.int16), before[0][pages, slots])
    # pages that do not exist: the ledger moves, their rows do not
    c = Cache(lens, 4, 2, d, F16)
    table = c.table_d.clone()
    table[0, 4] = 10 ** 6
    status.zero_()
    m, t = ledger(3, 2, 32, seed=4)
    m[0, :, 16:20], m[0, :, :8] = 100.0, 0.5
    K.cache_evict(c.k, c.v, table, c.lens, m, t, 8, status=status)
    assert status.item() == K.STATUS_BAD_PAGE and (m[0, :, :8] == 100.0).sum() == 8
    K.cache_evict(c.k, c.v, table[:0], c.lens[:0], m[:0], t[:0], 8)      # no sequences


def test_weights_and_evictions_at_once():
    """Two streams, each with a batch of its own, give what each gives alone."""
    sides = [torch.cuda.Stream() for _ in range(2)]
    sets = []
    for i, dtype in enumerate((F16, BF16)):
        c = Cache([700, 90, 1500, 3], 16, 2, 128, dtype, seed=i)
        q, lse = randn(4, 8, 128, seed=i), None
        lse = lse_of(c, q, 128 ** -0.5)
        m, t = ledger(4, 2, 1500, seed=i)
        want_m = K.attention_mass(q, c.k, c.table_d, c.lens, lse, m, out=m.clone())
        k0 = c.k.clone()
        alone = (torch.zeros(4, 2, 64, device="cuda"), torch.zeros(4, 2, 64, dtype=torch.int32,
                                                                   device="cuda"))
        K.cache_evict(*c.args, c.lens, want_m, t, 64, 8, *alone, torch.empty_like(c.lens))
        want_k = c.k.clone()
        sets.append((c, q, lse, m, t, want_m, k0, alone, want_k))
    for _ in range(5):
        got = []
        for c, *_, k0, _, _ in sets:
            c.k.copy_(k0)
        torch.cuda.synchronize()
        for side, (c, q, lse, m, t, want_m, _, alone, want_k) in zip(sides, sets):
            with torch.cuda.stream(side):
                x = K.attention_mass(q, c.k, c.table_d, c.lens, lse, m, out=m.clone())
                mo, ho = (torch.zeros_like(a) for a in alone)
                K.cache_evict(*c.args, c.lens, x, t, 64, 8, mo, ho, torch.empty_like(c.lens))
                got.append((x, mo, ho))
        torch.cuda.synchronize()
        for (x, mo, ho), (c, _, _, _, _, want_m, _, alone, want_k) in zip(got, sets):
            assert torch.equal(x, want_m) and torch.equal(mo, alone[0]) and torch.equal(ho, alone[1])
            assert torch.equal(c.k.view(torch.int16), want_k.view(torch.int16))


def test_evict_captured_and_other_stream():
    """One captured call serves later lengths, and runs where it is called."""
    hkv, d, keep = 2, 64, 32
    lens = [40, 33]
    m0, t0 = ledger(2, hkv, 64, seed=3)
    c = Cache([64, 64], 8, hkv, d, F16)
    m, t, n = m0.clone(), t0.clone(), i32(*lens)
    k0, v0 = c.k.clone(), c.v.clone()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        K.cache_evict(*c.args, i32(0, 0), m, t, keep, 4, max_len=64)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        K.cache_evict(*c.args, n, m, t, keep, 4, max_len=64)
    for lens in ([40, 33], [64, 5], [32, 50]):
        for x, y in ((m, m0), (t, t0), (c.k, k0), (c.v, v0)):
            x.copy_(y)
        n.copy_(i32(*lens))
        g.replay()
        moves = evict_plain(lens, m0.cpu(), t0.cpu(), keep, 4)
        wm, wk = m0.clone(), k0.clone()
        for (s, h), (a, b) in moves.items():
            if a:
                wm[s, h, b] = wm[s, h, a]
                wk[(*c.where(s, b), h)] = wk[(*c.where(s, a), h)]
        assert torch.equal(m, wm) and n.tolist() == [min(x, keep) for x in lens]
        assert torch.equal(c.k.view(torch.int16), wk.view(torch.int16))

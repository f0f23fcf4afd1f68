"""Rotary append, paged attention of single tokens, block-weight linear: each
against a plain 64-bit form, at the sizes and masks where it can go wrong, and
a decode step of all of them together."""
import math

import numpy as np
import pytest
import torch

from linuxnightmaresuite_b200 import _lib, kernels as K, synth
from linuxnightmaresuite_b200.attention import AttentionLayer, PagedKVCache
from linuxnightmaresuite_b200.moe_forward import MoELayer
from linuxnightmaresuite_b200.stacked import StackedMoE

from ._attention import (BF16, E4M3, F16, SCALES, Cache, attend, check_attention, check_linear,
                         check_stored, matrix, rotate)

pytestmark = pytest.mark.gpu


def randn(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).cuda()


# --------------------------------------------------------------------------- append

@pytest.mark.parametrize("dtype", [F16, BF16, E4M3])
@pytest.mark.parametrize("layout", ["nhd", "hnd"])
@pytest.mark.parametrize("hq,hkv,d,rot,interleaved,page", [
    (8, 2, 128, 128, False, 16),
    (4, 4, 64, 32, True, 5),        # partial, adjacent pairs, odd pages
    (3, 1, 80, 80, False, 1),       # rot / 2 = 40, one slot per page
    (5, 5, 256, 64, False, 64),
    (2, 1, 16, 6, False, 7),        # three pairs
    (1, 1, 16, 14, True, 3),
    (6, 3, 96, 0, False, 8),        # nothing turns
])
def test_append(dtype, layout, hq, hkv, d, rot, interleaved, page):
    lens = [page * 3 + 2, 1, 2 * page]
    c = Cache(lens, page, hkv, d, dtype, layout, seed=d)
    before = (c.k.clone().view(torch.uint8), c.v.clone().view(torch.uint8))
    seq = [0, 0, 0, 2, 1, 2, 0]
    pos = [lens[0] - 1, 0, page, 2 * page - 1, 0, page - 1, 2 * page]
    # q, k, v side by side, as the joint projection leaves them, with a gap
    qkv = randn(len(seq), (hq + 2 * hkv) * d + 4, seed=rot)
    q = qkv[:, :hq * d].unflatten(1, (hq, d))
    k = qkv[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
    v = qkv[:, (hq + hkv) * d:(hq + 2 * hkv) * d].unflatten(1, (hkv, d))
    freq = K.rope_inv_freq(rot, 10000.0) if rot else None
    p = torch.tensor(pos, dtype=torch.int32).cuda()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = K.rope_append(q, k, v, *c.args, p, freq, torch.tensor(seq, dtype=torch.int32).cuda(),
                        interleaved, status=status, **c.scales)
    f = freq if rot else torch.zeros(0, dtype=torch.float64, device="cuda")
    yq, bq = rotate(q.double(), p, f, interleaved)
    yk, bk = rotate(k.double(), p, f, interleaved)
    assert ((out.double() - yq).abs() <= bq).all()
    touched = torch.zeros(c.k.shape[:2], dtype=torch.bool, device="cuda")
    for i, (s, at) in enumerate(zip(seq, pos)):
        pages, slots = c.where(s, [at])
        touched[pages, slots] = True
        ks, vs = SCALES[dtype]
        check_stored(c.k[pages, slots][0], yk[i], bk[i], dtype, ks)
        check_stored(c.v[pages, slots][0], v[i].double(), 0 * bk[i], dtype, vs)
    for new, old in zip((c.k, c.v), before):        # every other slot as it was
        assert torch.equal(new.view(torch.uint8)[~touched], old[~touched])
    assert status.item() == 0


def test_append_in_place_and_far_positions():
    """q turned in place in the projection's output; positions where an f32
    angle would be off by whole radians."""
    T, hq, hkv, d, page = 4, 8, 2, 128, 16
    width = (1 << 24) // page
    c = Cache([page] * T, page, hkv, d, F16, width=width)
    pos = [(1 << 24) - 1, 1 << 20, 131071, 16777213]
    for s, p in enumerate(pos):
        c.table_d[s, p // page] = c.table[s, 0].item()
    qkv = randn(T, (hq + 2 * hkv) * d, seed=5)
    keep = qkv.clone()
    q, k, v = (qkv[:, a * d:b * d].unflatten(1, (b - a, d))
               for a, b in ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv)))
    p = torch.tensor(pos, dtype=torch.int32).cuda()
    freq = K.rope_inv_freq(d, 500000.0)
    got = K.rope_append(q, k, v, *c.args, p, freq, q_out=q)
    assert got.data_ptr() == qkv.data_ptr()
    y, bound = rotate(keep[:, :hq * d].unflatten(1, (hq, d)).double(), p, freq, False)
    assert ((q.double() - y).abs() <= bound).all()
    assert torch.equal(qkv[:, hq * d:], keep[:, hq * d:])


def test_append_skips_padding_and_reports_bad_pages():
    hkv, d, page = 2, 64, 4
    c = Cache([8, 8, 8, 8, 8], page, hkv, d, BF16)
    old_k, old_v = c.k.clone(), c.v.clone()
    table = c.table_d.clone()
    table[2, 1] = c.k.shape[0]                      # one past the pool
    table[3, 1] = -1
    q, k, v = randn(6, 4, d), randn(6, hkv, d, seed=1), randn(6, hkv, d, seed=2)
    out = torch.full_like(q, 7.0)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    #        padding, fine, bad page, bad page, behind the table, no such sequence
    pos = torch.tensor([-1, 5, 6, 7, page * table.shape[1], 0], dtype=torch.int32).cuda()
    seq = torch.tensor([0, 1, 2, 3, 4, 5], dtype=torch.int32).cuda()
    freq = K.rope_inv_freq(d)
    K.rope_append(q, k, v, c.k, c.v, table, pos, freq, seq, q_out=out, status=status)
    assert status.item() == K.STATUS_BAD_PAGE
    assert (out[0] == 7.0).all()
    y, bound = rotate(q[1:].double(), pos[1:], freq, False)
    assert ((out[1:].double() - y).abs() <= bound).all()
    pages, slots = c.where(1, [5])
    changed = torch.zeros(c.k.shape[:2], dtype=torch.bool, device="cuda")
    changed[pages, slots] = True
    for new, old in ((c.k, old_k), (c.v, old_v)):
        assert torch.equal(new[~changed].view(torch.int16), old[~changed].view(torch.int16))
    y, bound = rotate(k[1:2].double(), pos[1:2], freq, False)
    check_stored(c.k[pages, slots], y, bound, BF16, 1.0)
    status.zero_()                                  # all padding: nothing to report
    K.rope_append(q, k, v, c.k, c.v, table, torch.full_like(pos, -1), freq, seq, q_out=out,
                  status=status)
    assert status.item() == 0


def test_append_without_q_and_without_tokens():
    c = Cache([4, 4], 4, 1, 32, F16)
    k, v = randn(2, 1, 32), randn(2, 1, 32, seed=1)
    pos = torch.tensor([3, 0], dtype=torch.int32).cuda()
    assert K.rope_append(None, k, v, *c.args, pos) is None
    for s, at in ((0, 3), (1, 0)):
        pages, slots = c.where(s, [at])
        assert torch.equal(c.k[pages, slots][0], k[s].half())
        assert torch.equal(c.v[pages, slots][0], v[s].half())
    empty = K.rope_append(randn(0, 2, 32), k[:0], v[:0], *c.args, pos[:0])
    assert empty.shape == (0, 2, 32)


def test_append_saturates_and_keeps_nan():
    c = Cache([4], 4, 1, 16, E4M3)
    k = torch.zeros((1, 1, 16), device="cuda")
    k[0, 0, :6] = torch.tensor([1e9, -1e9, math.inf, -math.inf, math.nan, 1.0])
    pos = torch.tensor([2], dtype=torch.int32).cuda()
    K.rope_append(None, k, k, *c.args, pos, **c.scales)
    pages, slots = c.where(0, [2])
    got = c.k[pages, slots].float().view(-1)[:6].tolist()
    assert got[:4] == [448.0, -448.0, 448.0, -448.0] and math.isnan(got[4]) and got[5] == 32.0


# --------------------------------------------------------------------------- attention

@pytest.mark.parametrize("dtype", [F16, BF16, E4M3])
@pytest.mark.parametrize("layout", ["nhd", "hnd"])
@pytest.mark.parametrize("hq,hkv,d,page", [
    (8, 2, 128, 16),
    (16, 16, 64, 24),     # one query head per key head; pages end inside a tile
    (4, 1, 256, 7),       # odd pages
    (10, 2, 80, 1),       # five heads share one; one slot per page
    (3, 1, 96, 64),
    (16, 1, 128, 32),     # more heads than one group holds
    (40, 2, 64, 8),       # three groups of heads
    (7, 7, 16, 128),
    (2, 1, 192, 16),
])
def test_attention(dtype, layout, hq, hkv, d, page):
    lens = [1, 15, 16, 17, 0, 63, 64, 65, 129, 777, 31]
    c = Cache(lens, page, hkv, d, dtype, layout, seed=hq + d)
    q = 1.5 * randn(len(lens), hq, d, seed=3)
    ws = K.paged_attention_workspace(len(lens), hq, hkv, d, "cuda")
    out, lse = K.paged_attention(q, *c.args, c.lens, ws=ws, return_lse=True, **c.scales)
    assert K.read_status(ws) == 0
    check_attention(c, q, out, lse, d ** -0.5)
    assert (out[4] == 0).all()
    again, lse2 = K.paged_attention(q, *c.args, c.lens, ws=ws, return_lse=True, max_len=777,
                                    **c.scales)
    check_attention(c, q, again, lse2, d ** -0.5)
    third = K.paged_attention(q, *c.args, c.lens, ws=ws, max_len=777, **c.scales)
    assert torch.equal(third, again)               # equal calls, equal bits


@pytest.mark.parametrize("dtype", [F16, BF16, E4M3])
@pytest.mark.parametrize("window,cap,scale", [(1, 0.0, None), (16, 0.0, 0.3), (100, 30.0, None),
                                              (5000, 5.0, 1.0), (0, 50.0, 0.0), (0, 0.0, -0.2),
                                              (0, 0.0, 0.0), (64, 8.0, -1.0)])
def test_attention_window_cap_scale(dtype, window, cap, scale):
    hq, hkv, d, page = 6, 2, 128, 16
    lens = [1, 0, 99, 100, 101, 400, 1500]
    c = Cache(lens, page, hkv, d, dtype, seed=window)
    q = randn(len(lens), hq, d, seed=4)
    out, lse = K.paged_attention(q, *c.args, c.lens, scale=scale, window=window, softcap=cap,
                                 return_lse=True, **c.scales)
    check_attention(c, q, out, lse, d ** -0.5 if scale is None else scale, window, cap)


@pytest.mark.parametrize("dtype", [F16, BF16, E4M3])
@pytest.mark.parametrize("seqs,length,hq,hkv,d", [(1, 40001, 8, 2, 128), (3, 20000, 8, 1, 64),
                                                  (1, 30011, 4, 4, 256), (2, 9000, 16, 1, 128)])
def test_attention_long(dtype, seqs, length, hq, hkv, d):
    """Sequences that are split over many CTAs and joined."""
    lens = [length - 37 * s for s in range(seqs)]
    c = Cache(lens, 16, hkv, d, dtype, seed=length)
    q = 2.0 * randn(seqs, hq, d, seed=5)
    ws = K.paged_attention_workspace(seqs, hq, hkv, d, "cuda")
    first = None
    for _ in range(3):
        out, lse = K.paged_attention(q, *c.args, c.lens, ws=ws, return_lse=True, **c.scales)
        check_attention(c, q, out, lse, d ** -0.5)
        first = out if first is None else first
        assert torch.equal(out, first)
    assert K.read_status(ws) == 0


def test_attention_large_scores_and_one_key():
    """Scores in the hundreds: only the maximum's key counts; a single key
    gives its value whatever its score."""
    hq, hkv, d = 4, 2, 128
    c = Cache([600, 1], 16, hkv, d, F16, seed=9)
    q = 60.0 * randn(2, hq, d, seed=6)
    out, lse = K.paged_attention(q, *c.args, c.lens, return_lse=True)
    check_attention(c, q, out, lse, d ** -0.5)
    torch.testing.assert_close(out[1], c.vd[1][0].repeat_interleave(2, 0).float(), rtol=1e-6,
                               atol=1e-6)


@pytest.mark.parametrize("scale", [1e-30, 3e-12, 1.0, 1e6, 1e25])
def test_attention_q_of_any_size(scale):
    """Rows of q far from 1 (undone by the score scale) lose nothing."""
    hq, hkv, d = 8, 2, 64
    for dtype in (F16, BF16):
        c = Cache([70, 300], 16, hkv, d, dtype, seed=10)
        q = randn(2, hq, d, seed=7) * scale
        out = K.paged_attention(q, *c.args, c.lens, scale=0.125 / scale)
        check_attention(c, q, out, None, float(np.float32(0.125 / scale)))


def test_attention_strided_q_and_padding_rows():
    """q as a slice of the projection's output; sequences behind the batch
    have length 0 and no pages."""
    hq, hkv, d = 8, 4, 64
    lens = [50, 3, 0, 0]
    c = Cache(lens, 16, hkv, d, BF16, seed=11)
    qkv = randn(4, (hq + 2 * hkv) * d, seed=8)
    qkv[2:] = math.nan
    q = qkv[:, :hq * d].unflatten(1, (hq, d))
    out, lse = K.paged_attention(q, *c.args, c.lens, return_lse=True)
    check_attention(c, q, out, lse, d ** -0.5)
    neg = torch.tensor([50, 3, -1, -5], dtype=torch.int32).cuda()
    out2, lse2 = K.paged_attention(q, *c.args, neg, return_lse=True)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)


def test_attention_bad_pages_and_lengths():
    """A page that does not exist is left out and reported; so is a length
    that the table does not hold."""
    hq, hkv, d, page = 4, 2, 64, 16
    c = Cache([64, 40], page, hkv, d, F16, seed=12, width=4)
    q = randn(2, hq, d, seed=9)
    ws = K.paged_attention_workspace(2, hq, hkv, d, "cuda")
    for bad in (c.k.shape[0], -1, 2 ** 30):
        table = c.table_d.clone()
        table[0, 1] = bad
        out = K.paged_attention(q, c.k, c.v, table, c.lens, ws=ws)
        assert K.read_status(ws) == K.STATUS_BAD_PAGE
        keep = [i for i in range(64) if i // page != 1]
        o, _, tol, _ = attend(q[0].double(), c.kd[0][keep], c.vd[0][keep], d ** -0.5)
        assert ((out[0].double() - o).abs() <= tol).all()
        o, _, tol, _ = attend(q[1].double(), c.kd[1], c.vd[1], d ** -0.5)
        assert ((out[1].double() - o).abs() <= tol).all()
    longer = torch.tensor([1000, 40], dtype=torch.int32).cuda()
    out = K.paged_attention(q, *c.args, longer, ws=ws)
    assert K.read_status(ws) == K.STATUS_BAD_PAGE
    check_attention(c, q, out, None, d ** -0.5)
    # every page of a sequence gone: nothing to attend to
    table = c.table_d.clone()
    table[0] = -1
    out, lse = K.paged_attention(q, c.k, c.v, table, c.lens, ws=ws, return_lse=True)
    assert K.read_status(ws) == K.STATUS_BAD_PAGE
    assert (out[0] == 0).all() and torch.isneginf(lse[0]).all()


def test_attention_infinite_keys_in_masked_slots():
    """Inf and NaN behind the end and before the window are never met."""
    hq, hkv, d, page = 4, 2, 64, 16
    for fill in (math.inf, -math.inf, math.nan):
        c = Cache([30], page, hkv, d, F16, seed=13, fill=fill)
        pages, slots = c.where(0, range(20))
        c.k[pages, slots] = fill
        c.v[pages, slots] = fill
        q = randn(1, hq, d, seed=10)
        out = K.paged_attention(q, *c.args, c.lens, window=10)
        check_attention(c, q, out, None, d ** -0.5, 10)


def test_attention_offsets_past_32_bits():
    """Pages whose elements lie behind 2^31 and 2^32 in the pool."""
    hkv, d, page = 8, 128, 64
    per = page * hkv * d
    total = (1 << 32) // per + 40
    k = torch.empty((total, page, hkv, d), dtype=E4M3, device="cuda")
    v = torch.empty_like(k)
    c = Cache([100, 200], page, hkv, d, E4M3, seed=14)
    home = {}
    for i in sorted(set(c.table.flatten().tolist()) - {-7}):
        home[i] = total - 1 - i if i % 2 else (1 << 31) // per + i
        k[home[i]].copy_(c.k[i])
        v[home[i]].copy_(c.v[i])
    table = torch.tensor([[home.get(x, -7) for x in row] for row in c.table.tolist()],
                         dtype=torch.int32).cuda()
    q = randn(2, 16, d, seed=11)
    out = K.paged_attention(q, k, v, table, c.lens, **c.scales)
    check_attention(c, q, out, None, d ** -0.5)
    kn, vn = randn(2, hkv, d, seed=12), randn(2, hkv, d, seed=13)
    pos = torch.tensor([99, 199], dtype=torch.int32).cuda()
    K.rope_append(None, kn, vn, k, v, table, pos, **c.scales)
    for s, p in ((0, 99), (1, 199)):
        at = home[c.table[s, p // page].item()]
        check_stored(k[at, p % page], kn[s].double(), 0 * kn[s].double(), E4M3, c.k_scale)
        check_stored(v[at, p % page], vn[s].double(), 0 * vn[s].double(), E4M3, c.v_scale)


@pytest.mark.parametrize("dtype", [F16, E4M3])
def test_other_cache_layouts(dtype):
    """Keys and values side by side in one pool, rows with padding behind them,
    a pool of one page, one slot per page, one key head."""
    hq, hkv, d = 4, 2, 64
    c = Cache([70, 33], 16, hkv, d, dtype, seed=20)
    q = randn(2, hq, d, seed=20)
    want = K.paged_attention(q, *c.args, c.lens, **c.scales)
    check_attention(c, q, want, None, d ** -0.5)
    bits = torch.uint8
    pool = torch.zeros((c.k.shape[0], 2) + c.k.shape[1:], dtype=dtype, device="cuda")
    pool.view(bits)[:, 0], pool.view(bits)[:, 1] = c.k.view(bits), c.v.view(bits)
    got = K.paged_attention(q, pool[:, 0], pool[:, 1], c.table_d, c.lens, **c.scales)
    assert torch.equal(got, want)
    wide = [torch.zeros(c.k.shape[:3] + (d + 16,), dtype=dtype, device="cuda") for _ in range(2)]
    for w, x in zip(wide, (c.k, c.v)):
        w.view(bits)[..., :x.view(bits).shape[-1]] = x.view(bits)
    got = K.paged_attention(q, wide[0][..., :d], wide[1][..., :d], c.table_d, c.lens, **c.scales)
    assert torch.equal(got, want)
    kn, vn, pos = randn(2, hkv, d, seed=21), randn(2, hkv, d, seed=22), c.lens - 1
    K.rope_append(None, kn, vn, *c.args, pos, **c.scales)
    for k, v in ((pool[:, 0], pool[:, 1]), (wide[0][..., :d], wide[1][..., :d])):
        K.rope_append(None, kn, vn, k, v, c.table_d, pos, **c.scales)
        assert torch.equal(k.contiguous().view(bits), c.k.view(bits))
        assert torch.equal(v.contiguous().view(bits), c.v.view(bits))
    one = Cache([5], 8, 1, d, dtype, seed=23, spare=0)
    out = K.paged_attention(q[:1], *one.args, one.lens, **one.scales)
    check_attention(one, q[:1], out, None, d ** -0.5)
    single = Cache([1], 1, 1, d, dtype, seed=24, spare=0)
    out = K.paged_attention(q[:1], *single.args, single.lens, **single.scales)
    check_attention(single, q[:1], out, None, d ** -0.5)
    odd = torch.zeros((3, 16 * (2 * d + 16)), dtype=dtype, device="cuda").as_strided(
        (3, 16, 2, d), (16 * (2 * d + 16), 2 * d + 16, d, 1))
    with pytest.raises(_lib.MoEError, match="strides"):
        K.paged_attention(q, odd, odd, c.table_d, c.lens, **c.scales)


def test_pages_shared_by_sequences():
    """A common prefix is held once; two sequences list its pages."""
    hq, hkv, d, page = 8, 2, 128, 16
    c = Cache([64, 30], page, hkv, d, BF16, seed=25)
    table = c.table_d.clone()
    table[1, 2] = table[1, 0]
    table[1, 3] = table[1, 1]
    table[1, 0], table[1, 1] = table[0, 0], table[0, 1]
    lens = torch.tensor([64, 62], dtype=torch.int32).cuda()
    q = randn(2, hq, d, seed=26)
    out = K.paged_attention(q, c.k, c.v, table, lens, max_len=1)   # too small a hint: still whole
    both = type("C", (), dict(kd=[c.kd[0], torch.cat([c.kd[0][:32], c.kd[1]])],
                              vd=[c.vd[0], torch.cat([c.vd[0][:32], c.vd[1]])]))
    check_attention(both, q, out, None, d ** -0.5)


def test_two_calls_at_once():
    """Two streams, a workspace each, many calls under way together."""
    hq, hkv, d = 8, 2, 128
    caches = [Cache([6000, 10], 16, hkv, d, F16, seed=30 + i) for i in range(2)]
    qs = [randn(2, hq, d, seed=32 + i) for i in range(2)]
    ws = [K.paged_attention_workspace(2, hq, hkv, d, "cuda") for _ in range(2)]
    want = [K.paged_attention(q, *c.args, c.lens, ws=w) for q, c, w in zip(qs, caches, ws)]
    rng = np.random.default_rng(3)
    raw, w, big = matrix(rng, 2, 512, 4096)
    lw = K.LinearWeights(torch.from_numpy(raw.reshape(-1)).cuda(), 2, 512, 4096)
    xs = [randn(3 + 8 * i, 4096, seed=34 + i) for i in range(2)]
    want_y = [K.linear(x, lw) for x in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((K.paged_attention(qs[i], *caches[i].args, caches[i].lens, ws=ws[i]),
                               K.linear(xs[i], lw)))
    torch.cuda.synchronize()
    for i in range(2):
        for o, y in got[i]:
            assert torch.equal(o, want[i]) and torch.equal(y, want_y[i])


def test_attention_many_sequences():
    """More sequences than a CTA has threads, most of them empty."""
    hq, hkv, d = 4, 2, 64
    lens = [(s * 37) % 90 if s % 3 == 0 else 0 for s in range(1500)]
    c = Cache(lens, 16, hkv, d, F16, seed=15)
    q = randn(len(lens), hq, d, seed=14)
    out, lse = K.paged_attention(q, *c.args, c.lens, return_lse=True)
    check_attention(c, q, out, lse, d ** -0.5)


@pytest.mark.parametrize("dtype", [F16, BF16, E4M3])
@pytest.mark.parametrize("hq,hkv,d", [(5, 1, 128), (8, 8, 64), (6, 3, 256), (24, 2, 96)])
def test_attention_parts_of_two_units(dtype, hq, hkv, d):
    """Runs that begin in one unit and end in another, each joined by whichever
    CTA comes last: the same bits every time."""
    lens = [4001, 4733, 0, 1, 5099, 3777, 4510]
    c = Cache(lens, 16, hkv, d, dtype, seed=d)
    q = randn(len(lens), hq, d, seed=3)
    ws = K.paged_attention_workspace(len(lens), hq, hkv, d, "cuda")
    out, lse = K.paged_attention(q, *c.args, c.lens, return_lse=True, ws=ws,
                                 **c.scales)
    check_attention(c, q, out, lse, d ** -0.5)
    for _ in range(50):
        again, l2 = K.paged_attention(q, *c.args, c.lens, return_lse=True, ws=ws, **c.scales)
        assert torch.equal(again, out) and torch.equal(l2, lse)


def test_attention_captured_and_replayed_with_other_lengths():
    """One captured launch serves every later length; two captured graphs
    that share a workspace replay in turn."""
    hq, hkv, d = 8, 2, 128
    lens = [5000, 40, 0]
    c = Cache(lens, 16, hkv, d, F16, seed=16)
    q = randn(3, hq, d, seed=15)
    n = c.lens.clone()
    ws = K.paged_attention_workspace(3, hq, hkv, d, "cuda")
    outs = [torch.empty_like(q), torch.empty_like(q)]
    K.paged_attention(q, *c.args, n, ws=ws, out=outs[0])
    graphs = []
    for o, w in zip(outs, (0, 64)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            K.paged_attention(q, *c.args, n, ws=ws, out=o, window=w)
        graphs.append(g)
    for new in (lens, [17, 0, 0], [4999, 40, 0], [1, 1, 0]):
        n.copy_(torch.tensor(new, dtype=torch.int32))
        for o in outs:
            o.fill_(math.nan)
        for g in graphs:
            g.replay()
        cut = type("C", (), dict(kd=[x[:m] for x, m in zip(c.kd, new)],
                                 vd=[x[:m] for x, m in zip(c.vd, new)]))
        check_attention(cut, q, outs[0], None, d ** -0.5)
        check_attention(cut, q, outs[1], None, d ** -0.5, 64)


def test_operators_on_another_stream():
    hq, hkv, d = 8, 2, 128
    c = Cache([900], 16, hkv, d, F16, seed=17)
    q = randn(1, hq, d, seed=16)
    rng = np.random.default_rng(0)
    raw, w, big = matrix(rng, 2, 96, 128)
    lw = K.LinearWeights(torch.from_numpy(raw.reshape(-1)).cuda(), 2, 96, 128)
    x = randn(2, 128, seed=17)
    want, want_y = K.paged_attention(q, *c.args, c.lens), K.linear(x, lw)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got, y = K.paged_attention(q, *c.args, c.lens), K.linear(x, lw)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(y, want_y)


# --------------------------------------------------------------------------- linear

@pytest.mark.parametrize("qtype", [2, 8])
@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 8, 11, 16, 17, 37])
@pytest.mark.parametrize("rows,cols", [(16, 64), (1, 32), (17, 96), (203, 1056), (96, 4128)])
def test_linear(qtype, T, rows, cols):
    rng = np.random.default_rng(rows + T)
    raw, w, big = matrix(rng, qtype, rows, cols)
    lw = K.LinearWeights(torch.from_numpy(raw.reshape(-1)).cuda(), qtype, rows, cols)
    x = rng.standard_normal((T, cols), dtype=np.float32)
    y = K.linear(torch.from_numpy(x).cuda(), lw)
    check_linear(y.cpu().numpy(), x, w, big)
    assert torch.equal(K.linear(torch.from_numpy(x).cuda(), lw), y)


@pytest.mark.parametrize("qtype", [2, 8])
@pytest.mark.parametrize("T,rows,cols", [(1, 6144, 2816), (1, 20011, 1024), (4, 2816, 8192),
                                         (16, 4096, 8192), (9, 513, 12288), (1, 64, 32768),
                                         (16, 64, 32768), (33, 1024, 2816), (6, 40000, 512), (3, 40, 32768),
                                         (7, 33, 32768)])
def test_linear_wide(qtype, T, rows, cols):
    rng = np.random.default_rng(cols)
    raw, w, big = matrix(rng, qtype, rows, cols)
    lw = K.LinearWeights(torch.from_numpy(raw.reshape(-1)).cuda(), qtype, rows, cols)
    x = rng.standard_normal((T, cols), dtype=np.float32)
    res = rng.standard_normal((T, rows), dtype=np.float32)
    y = K.linear(torch.from_numpy(x).cuda(), lw, residual=torch.from_numpy(res).cuda())
    check_linear(y.cpu().numpy(), x, w, big, res)


@pytest.mark.parametrize("qtype", [2, 8])
@pytest.mark.parametrize("T,rows,cols", [(16, 20011, 4096), (8, 20011, 4096), (1, 20011, 4096),
                                         (13, 65541, 512), (3, 9003, 2848)])
def test_linear_several_rounds(qtype, T, rows, cols):
    """More rows than the GPU takes at a time, alone and in clusters, in place."""
    rng = np.random.default_rng(rows + cols)
    raw, w, big = matrix(rng, qtype, rows, cols)
    lw = K.LinearWeights(torch.from_numpy(raw.reshape(-1)).cuda(), qtype, rows, cols)
    x = rng.standard_normal((T, cols), dtype=np.float32)
    res = rng.standard_normal((T, rows), dtype=np.float32)
    y, xd = torch.from_numpy(res).cuda(), torch.from_numpy(x).cuda()
    K.linear(xd, lw, residual=y, out=y)
    check_linear(y.cpu().numpy(), x, w, big, res)
    for _ in range(20):
        assert torch.equal(K.linear(xd, lw, residual=torch.from_numpy(res).cuda()), y)


@pytest.mark.parametrize("T", [1, 2, 7])
def test_linear_widest(T):
    """Columns that leave room for fewer rows and tiles at a time, and more
    than fit at all."""
    rng = np.random.default_rng(7)
    raw, w, big = matrix(rng, 2, 40, 65536)
    lw = K.LinearWeights(torch.from_numpy(raw.reshape(-1)).cuda(), 2, 40, 65536)
    x = rng.standard_normal((T, 65536), dtype=np.float32)
    check_linear(K.linear(torch.from_numpy(x).cuda(), lw).cpu().numpy(), x, w, big)
    for qtype in (2, 8):
        wide = K.LinearWeights(torch.zeros(16 * (1 << 20) // 32 * synth.block_bytes(qtype),
                                           dtype=torch.uint8, device="cuda"), qtype, 16, 1 << 20)
        with pytest.raises(_lib.MoEError, match="do not fit"):
            K.linear(torch.zeros((T, 1 << 20), device="cuda"), wide)


def test_linear_many_rows():
    """More rows than one pass, the last pass with one of them."""
    rng = np.random.default_rng(5)
    raw, w, big = matrix(rng, 2, 80, 224)
    lw = K.LinearWeights(torch.from_numpy(raw.reshape(-1)).cuda(), 2, 80, 224)
    x = rng.standard_normal((321, 224), dtype=np.float32)
    y = K.linear(torch.from_numpy(x).cuda(), lw).cpu().numpy()
    check_linear(y, x, w, big)
    # parts of the batch by themselves
    for t in (0, 15, 16, 320):
        one = K.linear(torch.from_numpy(x[t:t + 16]).cuda(), lw).cpu().numpy()
        check_linear(one, x[t:t + 16], w, big)


def test_linear_captured():
    rng = np.random.default_rng(6)
    raw, w, big = matrix(rng, 2, 256, 8192)
    lw = K.LinearWeights(torch.from_numpy(raw.reshape(-1)).cuda(), 2, 256, 8192)
    for T in (1, 2, 16):
        x = torch.zeros((T, 8192), device="cuda")
        y = torch.empty((T, 256), device="cuda")
        K.linear(x, lw, out=y)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            K.linear(x, lw, out=y)
        for seed in range(3):
            x.copy_(randn(T, 8192, seed=seed))
            g.replay()
            check_linear(y.cpu().numpy(), x.cpu().numpy(), w, big)


def test_linear_strides_residual_in_place_and_no_rows():
    rng = np.random.default_rng(1)
    rows, cols, T = 100, 160, 6
    raw, w, big = matrix(rng, 2, rows, cols)
    lw = K.LinearWeights(torch.from_numpy(raw.reshape(-1)).cuda(), 2, rows, cols)
    wide = randn(T, cols + 37, seed=3)
    wide[:, :1] = math.nan                          # an odd offset into rows of an odd stride
    x = wide[:, 1:cols + 1]
    buf = randn(T, rows + 11, seed=4)
    keep = buf.clone()
    got = K.linear(x, lw, residual=buf[:, 3:rows + 3], out=buf[:, 3:rows + 3])
    assert got.data_ptr() == buf[:, 3:].data_ptr()
    check_linear(got.cpu().numpy(), x.cpu().numpy(), w, big, keep[:, 3:rows + 3].cpu().numpy())
    assert torch.equal(buf[:, :3], keep[:, :3]) and torch.equal(buf[:, rows + 3:],
                                                               keep[:, rows + 3:])
    assert K.linear(x[:0], lw).shape == (0, rows)
    one = x[:1].expand(3, cols)                     # one row for every token (stride 0)
    y = K.linear(one, lw)
    assert torch.equal(y[0], y[1]) and torch.equal(y[0], y[2])


def test_linear_special_values():
    """Rows of zeros, of huge and of tiny values; Inf and NaN stay in their row."""
    rng = np.random.default_rng(2)
    rows, cols = 64, 256
    raw, w, big = matrix(rng, 2, rows, cols)
    lw = K.LinearWeights(torch.from_numpy(raw.reshape(-1)).cuda(), 2, rows, cols)
    x = rng.standard_normal((6, cols), dtype=np.float32)
    x[0] = 0
    x[1] *= 1e30
    x[2] *= 1e-30
    x[3, 7] = np.inf
    x[4, 9] = np.nan
    y = K.linear(torch.from_numpy(x).cuda(), lw).cpu().numpy()
    assert (y[0] == 0).all()
    good = [0, 1, 2, 5]
    check_linear(y[good], x[good], w, big)
    assert not np.isfinite(y[3]).any() and np.isnan(y[4]).all()


# --------------------------------------------------------------------------- together

def _decoder(dtype, qtype, layers=2, window=0):
    dev = torch.device("cuda:0")
    cfg = synth.MoEConfig("decoder", 512, 8, 2, 256, 4, synth.QTYPE_Q4_0, 0.01)
    hq, hkv, d = 8, 2, 64
    rng = np.random.default_rng(21)
    moe, norms, att, att_norms, mats = [], [], [], [], []
    for li in range(layers):
        data = synth.make_layer_device(cfg, 31, 4, 0, cfg.n_experts, dev, layer=li)
        moe.append(MoELayer.from_blocks(data.gate_w, data.w_gate, data.w_up, data.w_down,
                                        cfg.qtype, cfg.top_k, mode=cfg.route_mode, device=dev))
        norms.append(torch.from_numpy(data.norm_w).to(dev))
        w = [matrix(rng, qtype, r, c, 0.003 if qtype == 2 else 0.0006)
             for r, c in ((hq * d, 512), (hkv * d, 512), (hkv * d, 512), (512, hq * d))]
        att.append(AttentionLayer.from_blocks(*(m[0].reshape(-1) for m in w), qtype, 512, hq, hkv,
                                              d, window=window, device=dev))
        att_norms.append(torch.from_numpy(
            (1 + 0.1 * rng.standard_normal(512)).astype(np.float32)).to(dev))
        mats.append([torch.from_numpy(m[1]).to(dev) for m in w])
    return StackedMoE(moe, norms, attention=att, attention_norms=att_norms), mats


@pytest.mark.parametrize("dtype,qtype,window", [(F16, 2, 0), (BF16, 8, 6), (E4M3, 2, 0)])
def test_decode_steps(dtype, qtype, window):
    """Decoder layers over a growing cache, sequences joining and leaving:
    every attention sub-layer against its 64-bit form on the step's own input
    and the cache's own contents, every step against the layers one by one."""
    dev = torch.device("cuda:0")
    hq, hkv, d, S = 8, 2, 64, 3
    stack, mats = _decoder(dtype, qtype, window=window)
    ks, vs = SCALES[dtype]
    caches, alone = ([PagedKVCache(24, 4, hkv, d, S, 6, dtype, ks, vs, dev) for _ in range(2)]
                     for _ in range(2))
    joins, leaves = [0, 3, 5], [17, 11, 17]
    freq = K.rope_inv_freq(d)
    for step in range(17):
        pos = [step - a if a <= step < b else -1 for a, b in zip(joins, leaves)]
        for s, p in enumerate(pos):
            for c in caches + alone:
                c.reserve(s, p + 1)
                if p < 0 and step >= leaves[s]:
                    c.release(s)
        positions = torch.tensor(pos, dtype=torch.int32, device=dev)
        lens = positions + 1
        x = randn(S, 512, seed=100 + step)
        y = stack.forward(x, caches=caches, positions=positions, seq_lens=lens)
        cur = x.clone()
        for i in range(2):
            xn = K.rms_norm(cur, stack.attention_norms[i], stack.eps)
            nxt = stack.attention[i].forward(xn, alone[i], positions, lens, residual=cur)
            wq, wk, wv, wo = mats[i]
            for s, p in enumerate(pos):
                if p < 0:
                    assert torch.equal(nxt[s], cur[s])          # nothing attended: residual
                    continue
                q = (wq @ xn[s].double()).view(1, hq, d)
                q, _ = rotate(q, positions[s:s + 1], freq, False)
                t = torch.arange(p + 1, device=dev)
                pages = alone[i].block_table[s][t // 4].long()
                kd = alone[i].k[pages, t % 4].double() * ks
                vd = alone[i].v[pages, t % 4].double() * vs
                kn, _ = rotate((wk @ xn[s].double()).view(1, hkv, d), positions[s:s + 1], freq,
                               False)
                step_of = torch.finfo(dtype).eps        # a whole step: the f32 side may tip it
                assert ((kd[-1] - kn[0]).abs() <= kn[0].abs() * step_of + ks * 2.0 ** -9).all()
                o, _, to, _ = attend(q[0], kd, vd, d ** -0.5, window)
                want = wo @ o.reshape(-1) + cur[s].double()
                # q itself is off by f32 roundings of its projection (2^-18 of |q| in norm)
                tol = wo.abs() @ (to + 2.0 ** -16 * vd.abs().amax()).reshape(-1) + 1e-5
                assert ((nxt[s].double() - want).abs() <= tol).all()
            cur = stack.layers[i].forward_batch(K.rms_norm(nxt, stack.norms[i], stack.eps),
                                                residual=nxt)
        assert torch.equal(cur, y)
    for c in caches:
        assert c.device_status() == 0
    for a in stack.attention:
        assert a.device_status() == 0
    assert all(c.free_pages == 24 - 5 - 3 for c in caches)


def test_decode_step_captured():
    """The decoder step in a CUDA graph, positions advanced between replays."""
    dev = torch.device("cuda:0")
    stack, _ = _decoder(F16, 2)
    caches, eager = ([PagedKVCache(8, 8, 2, 64, 2, 4, F16, device=dev) for _ in range(2)]
                     for _ in range(2))
    for c in caches + eager:
        for s in range(2):
            c.reserve(s, 20)
    x = randn(2, 512, seed=1)
    pos = torch.zeros(2, dtype=torch.int32, device=dev)
    lens = pos + 1
    out = torch.empty_like(x)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        stack.forward(x, out=out, caches=caches, positions=pos, seq_lens=lens)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        stack.forward(x, out=out, caches=caches, positions=pos, seq_lens=lens)
    for step in range(20):
        x.copy_(randn(2, 512, seed=50 + step))
        pos.fill_(step)
        lens.fill_(step + 1)
        g.replay()
        want = stack.forward(x, caches=eager, positions=pos, seq_lens=lens)
        assert torch.equal(out, want), step


def test_refusals_on_the_device():
    c = Cache([8], 4, 2, 64, F16)
    q, k = randn(1, 4, 64), randn(1, 2, 64)
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    with pytest.raises(_lib.MoEError, match="head_dim"):
        bad = torch.zeros((2, 4, 2, 12), dtype=F16, device="cuda")
        K.paged_attention(randn(1, 4, 12), bad, bad, c.table_d, c.lens)
    with pytest.raises(_lib.MoEError, match="16 bytes"):
        bad = torch.zeros((2, 4, 2, 68), dtype=F16, device="cuda")[..., 4:]
        K.paged_attention(q, bad, bad, c.table_d, c.lens)
    with pytest.raises(_lib.MoEError, match="query heads"):
        K.paged_attention(randn(1, 3, 64), *c.args, c.lens)
    with pytest.raises(_lib.MoEError, match="workspace"):
        K.paged_attention(q, *c.args, c.lens, ws=torch.zeros(64, dtype=torch.uint8, device="cuda"))
    with pytest.raises(_lib.MoEError, match="scales"):
        K.paged_attention(q, *c.args, c.lens, k_scale=2.0)
    with pytest.raises(_lib.MoEError, match="rot"):
        K.rope_append(q, k, k, *c.args, pos, K.rope_inv_freq(66))
    with pytest.raises(_lib.MoEError, match="seq_ids"):
        K.rope_append(q.expand(2, 4, 64), k.expand(2, 2, 64), k.expand(2, 2, 64), *c.args,
                      pos.repeat(2))
    with pytest.raises(ValueError):
        K.paged_attention(randn(2, 4, 64), *c.args, c.lens)
    with pytest.raises(ValueError):
        K.paged_attention(q, c.k, c.v[:1], c.table_d, c.lens)
    with pytest.raises(TypeError):
        K.paged_attention(q.half(), *c.args, c.lens)
    with pytest.raises(TypeError):
        K.paged_attention(q, c.k.float(), c.v.float(), c.table_d, c.lens)
    raw = torch.zeros(18 * 2 * 16, dtype=torch.uint8, device="cuda")
    lw = K.LinearWeights(raw, 2, 16, 64)
    with pytest.raises(ValueError):
        K.linear(randn(1, 32), lw)
    with pytest.raises(ValueError):
        K.LinearWeights(raw, 2, 16, 32)
    with pytest.raises(ValueError):
        K.LinearWeights(raw, 12, 16, 64)

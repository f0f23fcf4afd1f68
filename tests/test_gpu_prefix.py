"""Attention of a batch that shares a prefix of pages, against the plain 64-bit
attention of each sequence over all of its keys."""
import math

import pytest
import torch

from linuxnightmaresuite_b200 import kernels as K

from ._attention import BF16, E4M3, F16, SCALES, Cache, attend
from .test_gpu_attention import randn

pytestmark = pytest.mark.gpu


class Shared:
    """Sequences of `own` tokens of their own behind a prefix of `pages` pages; own 0 with
    the prefix alone, None a padding row."""

    def __init__(self, own, pages, page, hkv, d, dtype, layout="nhd", seed=0):
        P = pages * page
        lens = [0 if n is None else P + n for n in own]
        self.c = c = Cache(lens + [P], page, hkv, d, dtype, layout, seed)
        self.pages = c.table_d[-1, :pages].contiguous()
        self.table = c.table_d[:-1].contiguous()
        self.table[:, :pages] = self.pages
        self.lens, self.P = c.lens[:-1].contiguous(), P
        for s, n in enumerate(lens):
            if n:
                c.kd[s], c.vd[s] = (torch.cat([x[-1], x[s][P:]]) for x in (c.kd, c.vd))
        self.kd, self.vd, self.dtype = c.kd[:-1], c.vd[:-1], dtype

    def call(self, q, form=K.PREFIX_TOGETHER, **kw):
        return K.prefix_attention(q, self.c.k, self.c.v, self.table, self.lens, self.pages,
                                  return_lse=True, form=form, **self.c.scales, **kw)

    def check(self, q, out, lse, scale, cap=0.0):
        """The bounds of `attend` (of its own 2^-20 for the accumulators 2^-19: 16 steps of a
        tile truncate, 2^-23 each), and for bf16 caches the probabilities' two parts: half a
        step, 2^-9, of what the first part leaves, 2^-9 of the value."""
        for s in range(q.shape[0]):
            o, l, to, tl = attend(q[s].double(), self.kd[s], self.vd[s], scale, 0, cap)
            if self.kd[s].shape[0] == 0:
                assert (out[s] == 0).all() and torch.isneginf(lse[s]).all()
                continue
            vmax = self.vd[s].abs().amax((0, 2)).repeat_interleave(q.shape[1] // self.vd[s].shape[1])
            to = to + vmax[:, None] * (2.0 ** -19 + (2.0 ** -18 if self.dtype == BF16 else 0.0))
            err = (out[s].double() - o).abs()
            assert (err <= to).all(), (s, err.max().item(), to.max().item())
            assert ((lse[s].double() - l).abs() <= tl + 2.0 ** -21).all(), s


@pytest.mark.parametrize("dtype", [F16, BF16, E4M3])
@pytest.mark.parametrize("own,pages,page,hq,hkv,d,layout", [
    ([1, 3], 1, 16, 4, 2, 128, "nhd"),              # less than a tile
    ([0, None, 37, 5], 8, 16, 8, 2, 128, "nhd"),    # one whole tile; nothing of one's own; padding
    ([2], 43, 7, 3, 1, 64, "hnd"),                  # odd pages: boxes of one row, a last tile of 45
    ([20, 1, 9], 5, 100, 16, 2, 256, "nhd"),
    ([0] * 35, 3, 128, 8, 2, 80, "nhd"),            # 140 rows: two row units
    ([1, 2], 400, 16, 16, 16, 96, "hnd"),           # runs that cross from head to head
    ([4] * 40, 21, 24, 16, 4, 192, "nhd"),          # column halves, the second one partly empty
    ([None, None, None], 2, 16, 2, 1, 128, "nhd"),  # nobody
    ([1, 1, 1], 300, 8, 5, 5, 16, "nhd"),
    ([30] * 6, 150, 64, 32, 8, 128, "nhd"),         # several tiles for each CTA
])
def test_prefix(dtype, own, pages, page, hq, hkv, d, layout):
    x = Shared(own, pages, page, hkv, d, dtype, layout, seed=hq + d)
    q = 1.5 * randn(len(own), hq, d, seed=3)
    ws = K.prefix_attention_workspace(len(own), hq, hkv, d, "cuda")
    out, lse = x.call(q, ws=ws, max_len=int(x.lens.max()))
    x.check(q, out, lse, d ** -0.5)
    assert K.read_status(ws) == 0
    again, lse2 = x.call(q, ws=ws, max_len=int(x.lens.max()))      # equal bits, and the workspace is ready
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("dtype", [F16, BF16, E4M3])
@pytest.mark.parametrize("d,hkv,pages,cap", [(256, 8, 100, 0.0), (192, 4, 390, 0.0), (128, 8, 110, 0.0),
                                             (128, 8, 110, 2.0), (64, 16, 60, 0.0), (64, 16, 60, 2.0)])
def test_prefix_next_head(dtype, d, hkv, pages, cap):
    """CTAs whose tiles go on with another head's rows: those are not fetched while products
    of the head before still read theirs, and each head has references of its own.  (Six calls:
    an order of warps that is wrong need not show in each.)"""
    x = Shared([2, 0, 1, 3, 2, 1], pages, 32, hkv, d, dtype, seed=d)
    q = 1.5 * randn(6, 4 * hkv, d, seed=7)
    q[:, ::3] *= 4                                   # rows, and so warps, that differ in their forms of tanh
    first = x.call(q, softcap=cap)
    x.check(q, *first, d ** -0.5, cap)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(x.call(q, softcap=cap), first))


@pytest.mark.parametrize("own,pages,together", [([5, 9], 4, False), ([3] * 64, 128, True)])
def test_prefix_form_by_size(own, pages, together):
    """Short prefixes and few sequences go one by one, the others together; equal bits of
    the form that is chosen."""
    x = Shared(own, pages, 16, 8, 128, F16)
    q = randn(len(own), 32, 128)
    got = x.call(q, K.PREFIX_AUTO)
    same = x.call(q, K.PREFIX_TOGETHER if together else K.PREFIX_EACH)
    assert torch.equal(got[0], same[0]) and torch.equal(got[1], same[1])
    other = x.call(q, K.PREFIX_EACH if together else K.PREFIX_TOGETHER)
    assert not torch.equal(got[0], other[0])
    for out, lse in (got, other):
        x.check(q, out, lse, 128 ** -0.5)


@pytest.mark.parametrize("dtype", [F16, BF16, E4M3])
def test_prefix_longer_than_some(dtype):
    """A sequence without the whole prefix is computed over the keys that it has."""
    x = Shared([3, 8, None, 0, 2], 10, 16, 2, 128, dtype)
    for s, n in ((1, 100), (3, 159), (4, 1)):
        x.lens[s] = n
        x.kd[s], x.vd[s] = x.kd[s][:n], x.vd[s][:n]
    # its pages need not be the prefix's
    x.table[1, :7] = x.c.table_d[1, :7]
    x.kd[1], x.vd[1] = (c[x.table[1, :7].long()].flatten(0, 1)[:100].double() * f
                        for c, f in ((x.c.k, x.c.k_scale), (x.c.v, x.c.v_scale)))
    q = randn(5, 8, 128)
    x.check(q, *x.call(q), 128 ** -0.5)


@pytest.mark.parametrize("dtype", [F16, BF16, E4M3])
def test_prefix_many_rows(dtype):
    """More row units than a team has members."""
    own = [s % 3 for s in range(300)]
    x = Shared(own, 20, 16, 2, 64, dtype, seed=5)
    q = randn(300, 16, 64, seed=6)
    x.check(q, *x.call(q), 0.125)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [F16, BF16, E4M3])
def test_prefix_scales_caps_strides(dtype, d):
    x = Shared([3, 0, None, 50], 30, 16, 2, d, dtype, seed=d)
    wide = randn(4, 8 * d + 3, seed=2)              # rows of q off 16 bytes
    q = wide[:, :8 * d].unflatten(1, (8, d))
    for cap, scale, up in ((0.0, 0.3, 1.0), (5.0, 0.5, 1.0), (30.0, -0.1, 1.0), (1e-6, 0.1, 1.0),
                           (0.0, 0.0, 1.0), (50.0, 1e-3, 1e4), (0.0, 1e30, 1e-31)):
        z = (q * up)
        if up == 1.0:
            z = q
        x.check(z, *x.call(z, scale=scale, softcap=cap), scale, cap)


def test_prefix_out_over_q_and_no_prefix():
    x = Shared([3, 8], 4, 16, 2, 64, F16)
    q = randn(2, 4, 64)
    want, lse = x.call(q)
    z = q.clone()
    got, lse2 = x.call(z, out=z)
    assert got is z and torch.equal(z, want) and torch.equal(lse, lse2)
    c = Cache([20, 7], 16, 2, 64, F16)
    a = K.paged_attention(q, *c.args, c.lens, return_lse=True)
    b = K.prefix_attention(q, *c.args, c.lens, x.pages[:0], return_lse=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_prefix_reports():
    x = Shared([3, 8, 2], 10, 16, 2, 128, F16)
    q = randn(3, 8, 128)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    x.lens[1] = 1 << 30                             # more than the table holds
    x.call(q, status=status)
    assert status.item() == K.STATUS_BAD_PAGE
    # a prefix page that does not exist is left out
    y = Shared([3, 8, 2], 10, 16, 2, 128, F16)
    for bad, at in ((-1, 2), (10 ** 6, 9)):
        y.pages[at] = bad
        status.zero_()
        out, lse = y.call(q, status=status)
        assert status.item() == K.STATUS_BAD_PAGE
    keep = torch.ones(160, dtype=torch.bool, device="cuda")
    keep[32:48], keep[144:] = False, False
    for s in range(3):
        n = torch.cat([keep, torch.ones(y.kd[s].shape[0] - 160, dtype=torch.bool, device="cuda")])
        y.kd[s], y.vd[s] = y.kd[s][n], y.vd[s][n]
    y.check(q, out, lse, 128 ** -0.5)


@pytest.mark.parametrize("dtype", [F16, BF16, E4M3])
def test_prefix_nan_beside_and_inf_within(dtype):
    """Slots behind the prefix's last page, or in a dropped one, may hold anything (the
    pools of these tests are NaN); a row of q that is NaN stays alone; an infinite value
    gives infinity or NaN in its column and nowhere else."""
    x = Shared([3, 8], 9, 16, 2, 64, dtype)
    q = randn(2, 4, 64)
    want, _ = x.call(q)
    z = q.clone()
    z[0, 1] = math.nan
    out, lse = x.call(z)
    assert torch.isnan(out[0, 1]).all() and torch.isnan(lse[0, 1])
    out[0, 1] = want[0, 1]
    assert torch.equal(out, want)
    if dtype != E4M3:
        x.c.v[x.pages[1].long(), 3, 0, 5] = math.inf
        out, _ = x.call(q)
        assert not torch.isfinite(out[:, :2, 5]).any()
        keep = torch.ones(64, dtype=torch.bool)
        keep[5] = False
        assert torch.equal(out[..., keep], want[..., keep]) and torch.equal(out[:, 2:], want[:, 2:])


def test_prefix_at_once_and_one_workspace_for_all_sizes():
    """Two streams with a workspace each; a workspace serves smaller batches and other heads'
    prefixes one after the other."""
    x, y = Shared([3] * 40, 60, 16, 2, 128, F16), Shared([9, 0, 7], 33, 16, 2, 128, BF16, seed=3)
    qx, qy = randn(40, 8, 128, seed=1), randn(3, 8, 128, seed=2)
    want_x, want_y = x.call(qx), y.call(qy)
    wide = K.prefix_attention_workspace(64, 8, 2, 128, "cuda")
    for _ in range(3):
        for s, q, want in ((x, qx, want_x), (y, qy, want_y)):
            got = s.call(q, ws=wide)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    spaces = [K.prefix_attention_workspace(40, 8, 2, 128, "cuda") for _ in range(2)]
    sides = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (s, q) in enumerate(((x, qx), (y, qy))):
            with torch.cuda.stream(sides[i]):
                got[i].append(s.call(q, ws=spaces[i]))
    torch.cuda.synchronize()
    for i, want in enumerate((want_x, want_y)):
        assert all(torch.equal(a, want[0]) and torch.equal(b, want[1]) for a, b in got[i])
    assert [K.read_status(w) for w in spaces + [wide]] == [0, 0, 0]


def test_prefix_captured_and_other_stream():
    """One captured call serves other lengths and pages."""
    x = Shared([3, 8, 60], 12, 16, 2, 128, F16)
    y = Shared([50, None, 0], 12, 16, 2, 128, F16, seed=4)
    q, ws = randn(3, 8, 128), K.prefix_attention_workspace(3, 8, 2, 128, "cuda")
    pool = (max(x.c.k.shape[0], y.c.k.shape[0]),) + x.c.k.shape[1:]
    k, v = (torch.full(pool, math.nan, dtype=F16, device="cuda") for _ in range(2))
    table = torch.full((3, max(x.table.shape[1], y.table.shape[1])), -1, dtype=torch.int32,
                       device="cuda")
    lens, pages = torch.zeros_like(x.lens), x.pages.clone()
    out = torch.empty_like(q)

    def call():
        return K.prefix_attention(q, k, v, table, lens, pages, out=out, return_lse=True, ws=ws,
                                  form=K.PREFIX_TOGETHER)[1]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        lse = call()
    for at, s in enumerate((x, y, x)):
        k[:s.c.k.shape[0]], v[:s.c.v.shape[0]] = s.c.k, s.c.v
        table[:, :s.table.shape[1]] = s.table
        lens.copy_(s.lens), pages.copy_(s.pages)
        q.copy_(randn(3, 8, 128, seed=at))
        out.fill_(math.nan)
        g.replay()
        s.check(q, out, lse, 128 ** -0.5)
    assert K.read_status(ws) == 0


@pytest.mark.parametrize("dtype,d", [(E4M3, 64), (E4M3, 16), (E4M3, 128), (F16, 64)])
def test_prefix_pages_missing_along_the_way(dtype, d):
    """Each CTA has some seventeen tiles, other keys of each are missing: which ones a tile has is
    known for eight tiles, and e4m3 heads of up to 64 come nearest to that.  (The bounds are those
    of the keys that are there.)"""
    pages, page = 5200, 8
    x = Shared([3, 0, 9], pages, page, 8, d, dtype, seed=11)
    g = torch.Generator().manual_seed(d)
    gone = torch.rand(pages, generator=g) < 0.03
    x.pages[gone.cuda()] = -1
    there = (~gone).repeat_interleave(page).cuda()
    for s in range(3):
        keep = torch.cat([there, torch.ones(x.kd[s].shape[0] - x.P, dtype=torch.bool, device="cuda")])
        x.kd[s], x.vd[s] = x.kd[s][keep], x.vd[s][keep]
    q = 1.5 * randn(3, 16, d, seed=4)
    first = x.call(q)
    x.check(q, *first, d ** -0.5)
    for _ in range(4):
        assert all(torch.equal(a, b) for a, b in zip(x.call(q), first))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [F16, BF16, E4M3])
def test_prefix_probabilities(dtype, d):
    """Each probability by itself: scores that are exact, a value of one for each of 16 keys in a
    column of its own.  Numerator and denominator are off by 2^-22 for exp2 each, the arguments
    (below 8 in magnitude: factor, reference and sum round) by 2^-22 each; the numerator's parts by
    2^-22, which two adds that truncate bring to 2^-21; the sum of 16 by 2^-20; quotient and scale
    by 2^-22 together."""
    x = Shared([0, 0, 0], 1, 16, 8, d, dtype, seed=d)
    page = int(x.pages[0])
    ks, vs = SCALES[dtype]
    k, v = (torch.zeros(16, 8, d, device="cuda") for _ in range(2))
    k[..., 0] = (4 * torch.rand(16, 8, generator=torch.Generator().manual_seed(d)) - 2).cuda() / ks
    v[range(16), :, range(16)] = 1.0
    x.c.k[page].copy_(k), x.c.v[page].copy_(v)
    kd = x.c.k[page].double() * ks
    q = torch.zeros(3, 16, d, device="cuda")
    q[..., 0] = torch.tensor([1.0, 0.5, -0.25], device="cuda")[:, None]
    out, _ = x.call(q, scale=1.0)
    s = torch.einsum("shd,nhd->shn", q.double(), kd.repeat_interleave(2, 1))
    want = torch.softmax(s, -1) * vs
    tol = 3 * 2.0 ** -21 + 2.0 ** -20 + 2.0 ** -21
    assert ((out[..., :16] - want).abs() <= want * tol).all(), ((out[..., :16] / want - 1).abs().max(), tol)
    assert (out[..., 16:] == 0).all()


@pytest.mark.parametrize("dtype", [F16, BF16, E4M3])
@pytest.mark.parametrize("d", [64, 256])
def test_prefix_and_own_keys_of_large_scores(dtype, d):
    """Scores that are all the same and exact, up to some thousands: the output is the share of
    own keys, whatever the scores.  Each weight is 2^7 but for the rounding of its argument, which
    is the same one everywhere; sums of 26 and of 160 equal terms and the join round a few
    times, 2^-24 each, exp2 of 0 and of -7 is exact: 2^-20."""
    x = Shared([26, 26, 0, 26, 26], 10, 16, 2, d, dtype, seed=d)
    ks, vs = SCALES[dtype]
    for cache in (x.c.k, x.c.v):
        cache.copy_(torch.zeros(cache.shape, device="cuda"))
    k = torch.zeros(16, 2, d, device="cuda")
    k[..., 0] = 14.0 / ks                           # 448 of e4m3
    one = torch.ones(16, 2, d, device="cuda")
    for page in x.table.flatten().unique().tolist():
        if page >= 0:
            x.c.k[page].copy_(k)
            if page not in x.pages.tolist():
                x.c.v[page].copy_(one)
    want = torch.tensor([n / (n + 160) for n in (26, 26, 0, 26, 26)], dtype=torch.float64).cuda() * vs
    for a in (1.0, 3.0, 9.25, 20.125, 66.625, 71.375, 150.75, 233.0, -66.625):
        q = torch.zeros(5, 4, d, device="cuda")
        q[..., 0] = a * torch.tensor([1.0, 1.25, 1.0, 1.5, 1.75], device="cuda")[:, None]
        out, lse = x.call(q, scale=1.0)
        err = (out - want[:, None, None]).abs()
        assert (err <= want[:, None, None] * 2.0 ** -20).all(), (a, (err / want[:, None, None]).nan_to_num().max())
        n = torch.tensor([186.0, 186.0, 160.0, 186.0, 186.0], dtype=torch.float64).cuda()
        s = 14.0 * q[..., 0].double()
        assert ((lse - s - n.log()[:, None]).abs() <= s.abs() * 2.0 ** -22 + 2.0 ** -20).all(), a


def test_prefix_out_off_16_bytes():
    """Refused where the forms go by the sizes; where the paged attention alone runs, taken."""
    x = Shared([3, 8], 4, 16, 2, 64, F16)
    q = randn(2, 4, 64)
    out = torch.empty(2 * 4 * 64 + 1, device="cuda")[1:].view(2, 4, 64)
    for form in (K.PREFIX_AUTO, K.PREFIX_TOGETHER):
        with pytest.raises(Exception, match="16-byte"):
            x.call(q, form, out=out)
    want = K.paged_attention(q, x.c.k, x.c.v, x.table, x.lens)
    assert torch.equal(x.call(q, K.PREFIX_EACH, out=out)[0], want)
    out.zero_()
    K.prefix_attention(q, x.c.k, x.c.v, x.table, x.lens, x.pages[:0], out=out)
    assert torch.equal(out, want)

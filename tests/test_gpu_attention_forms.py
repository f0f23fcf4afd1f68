"""Forms of the attention half's arguments that the documentation allows: odd
strides of single axes, heads and pages that share memory, status without a
workspace, infinities."""
import numpy as np
import pytest
import torch

from linuxnightmaresuite_b200 import _lib, kernels as K
from linuxnightmaresuite_b200.attention import PagedKVCache

from ._attention import BF16, E4M3, F16, Cache, check_attention, check_linear, matrix
from .test_gpu_attention import _decoder, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F16, E4M3])
def test_strides_of_single_axes(dtype):
    """One key head, one slot per page, one page: their strides count for nothing,
    in either cache."""
    d = 64
    for page, lens in ((16, [40, 3]), (1, [5, 2]), (64, [50])):
        c = Cache(lens, page, 1, d, dtype, seed=page, spare=0)
        q = randn(len(lens), 4, d, seed=page)
        want = K.paged_attention(q, *c.args, c.lens, **c.scales)
        check_attention(c, q, want, None, d ** -0.5)

        def odd(t, at):
            s = [t.stride(0), t.stride(1), at, 1]
            for i in (0, 1):
                if t.shape[i] == 1:
                    s[i] = at + i
            return t.as_strided(t.shape, s)
        k, v = odd(c.k, 3), odd(c.v, 5)
        assert torch.equal(K.paged_attention(q, k, v, c.table_d, c.lens, **c.scales), want)
        kn, pos = randn(len(lens), 1, d, seed=1), c.lens - 1
        K.rope_append(None, kn, kn, k, v, c.table_d, pos, **c.scales)
        got = c.k.view(torch.uint8).clone()
        K.rope_append(None, kn, kn, *c.args, pos, **c.scales)
        assert torch.equal(got, c.k.view(torch.uint8))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_heads_and_pages_that_share_memory(dtype):
    """The attention only reads: one head stands for all key heads, one page for all."""
    hkv, d, page = 4, 128, 16
    c = Cache([70, 33, 0], page, 1, d, dtype, seed=2)
    q = randn(3, 8, d, seed=2)
    k, v = (t.expand(-1, -1, hkv, -1) for t in (c.k, c.v))
    wide = type("C", (), dict(kd=[x.expand(-1, hkv, -1) for x in c.kd],
                              vd=[x.expand(-1, hkv, -1) for x in c.vd]))
    out, lse = K.paged_attention(q, k, v, c.table_d, c.lens, return_lse=True)
    check_attention(wide, q, out, lse, d ** -0.5)
    one = Cache([page], page, 1, d, dtype, seed=3, spare=0)
    k, v = (t.expand(5, -1, -1, -1) for t in (one.k, one.v))
    table = torch.tensor([[4, 0, 3, 1]], dtype=torch.int32).cuda()
    lens = torch.tensor([3 * page + 5], dtype=torch.int32).cuda()
    many = type("C", (), dict(kd=[one.kd[0].repeat(4, 1, 1)[:lens.item()]],
                              vd=[one.vd[0].repeat(4, 1, 1)[:lens.item()]]))
    out = K.paged_attention(q[:1], k, v, table, lens)
    check_attention(many, q[:1], out, None, d ** -0.5)
    for k, v in ((c.k.expand(-1, -1, hkv, -1),) * 2, (one.k.expand(5, -1, -1, -1),) * 2):
        new = torch.zeros((1, k.shape[2], d), device="cuda")
        with pytest.raises(_lib.MoEError, match="share memory"):
            K.rope_append(None, new, new, k, v, table, table[0, :1])
    with pytest.raises(_lib.MoEError, match="share memory"):
        t = c.k[:, :1].expand(-1, page, -1, -1)
        K.paged_attention(q, t, t, c.table_d, c.lens)


def test_status_without_a_workspace():
    """A page that does not exist is reported also where no workspace is kept."""
    cache = PagedKVCache(8, 4, 2, 64, max_seqs=2, dtype=F16)
    cache.reserve(0, 8)
    q, lens = randn(2, 4, 64), torch.tensor([8, 0], dtype=torch.int32).cuda()
    cache.attend(q, lens)
    assert cache.device_status() == 0
    lens[1] = 3                                     # no page was reserved
    cache.attend(q, lens)
    assert cache.device_status() == K.STATUS_BAD_PAGE
    assert cache.device_status() == 0
    ws = K.paged_attention_workspace(2, 4, 2, 64, "cuda")
    cache.attend(q, lens, ws=ws)                    # in the workspace, where one is given
    assert cache.device_status() == 0 and K.read_status(ws) == K.STATUS_BAD_PAGE
    for w in (None, ws):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        K.paged_attention(q, cache.k, cache.v, cache.block_table, lens, ws=w, status=status)
        assert status.item() == K.STATUS_BAD_PAGE
    with pytest.raises(TypeError):
        K.paged_attention(q, cache.k, cache.v, cache.block_table, lens, status=status.float())


@pytest.mark.parametrize("cap", [1e-44, 1e-38, 1e-30])
def test_smallest_cap(cap):
    """Scores capped to next to nothing, exact zeros among them: every key weighs
    the same."""
    c = Cache([50], 16, 2, 64, F16, seed=4)
    pages, slots = c.where(0, range(20, 30))
    c.k[pages, slots] = 0
    q = randn(1, 4, 64, seed=4)
    for size in (1.0, 1e30):
        out = K.paged_attention(size * q, *c.args, c.lens, softcap=cap)
        want = c.vd[0].mean(0).repeat_interleave(2, 0)
        assert (out[0].double() - want).abs().max() <= 2.0 ** -19 * c.vd[0].abs().max()


def test_no_sequences():
    """A batch without rows: nothing to do, and nothing wrong."""
    cache = PagedKVCache(4, 4, 2, 64, max_seqs=3, dtype=BF16)
    q, none = randn(0, 4, 64), torch.zeros(0, dtype=torch.int32, device="cuda")
    out, lse = cache.attend(q, none, return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    layer = _decoder(F16, 2, layers=1)[0].attention[0]
    y = layer.forward(randn(0, 512), PagedKVCache(4, 4, 2, 64, max_seqs=3), none, none)
    assert y.shape == (0, 512) and cache.device_status() == 0


def test_outputs_over_inputs():
    """x and the output side by side in one buffer; an output over its own input
    is refused before anything is written."""
    lw = K.LinearWeights(torch.randint(0, 255, (64 * 2 * 18,), dtype=torch.uint8).cuda(), 2, 64, 64)
    buf = randn(3, 128)
    keep = buf.clone()
    want = K.linear(keep[:, :64].contiguous(), lw)
    got = K.linear(buf[:, :64], lw, out=buf[:, 64:])
    assert torch.equal(got.view(torch.int32), want.view(torch.int32))    # NaN among the scales
    assert torch.equal(buf[:, :64], keep[:, :64])
    x = keep[:, :64].contiguous()
    for out in (x, buf.view(-1)[1:].as_strided((3, 64), (128, 1))):
        with pytest.raises(_lib.MoEError, match="overlap"):
            K.linear(x if out is x else buf[:, :64], lw, out=out)
    assert torch.equal(x, keep[:, :64])
    c = Cache([8, 8], 4, 2, 64, F16)
    q, k, pos = randn(2, 2, 64), randn(2, 2, 64, seed=1), c.lens - 1
    for out in (k, q.transpose(0, 1), q[:1].expand(2, 2, 64)):
        with pytest.raises(_lib.MoEError, match="q_out"):
            K.rope_append(q, k, k.clone(), *c.args, pos, K.rope_inv_freq(64), q_out=out)


@pytest.mark.parametrize("T", [1, 2, 4, 7, 16, 18])
@pytest.mark.parametrize("qtype,rows,cols", [(2, 40, 8192), (8, 67, 256)])
def test_linear_infinities(qtype, T, rows, cols):
    """Infinities and NaN give what the sum of the products gives, whatever the
    size of the row's other elements, and stay in their row."""
    rng = np.random.default_rng(T + cols)
    raw, w, big = matrix(rng, qtype, rows, cols)
    lw = K.LinearWeights(torch.from_numpy(raw.reshape(-1)).cuda(), qtype, rows, cols)
    for shift in range(6):
        x = rng.standard_normal((T, cols), dtype=np.float32)
        special = np.zeros(T, dtype=bool)
        for t in range(T):
            kind = (t + shift) % 6
            special[t] = kind != 0
            at = rng.integers(0, cols, 3)
            if kind == 1:
                x[t, at[0]] = np.inf
            elif kind == 2:
                x[t] *= np.float32(1e30)
                x[t, at[0]] = -np.inf
            elif kind == 3:
                x[t, at[:2]] = np.inf, -np.inf
            elif kind == 4:
                x[t] *= np.float32(1e-30)
                x[t, at] = np.inf
            elif kind == 5:
                x[t, at[:2]] = np.nan, np.inf
        y = K.linear(torch.from_numpy(x).cuda(), lw).cpu().numpy()
        with np.errstate(invalid="ignore"):
            want = (x.astype(np.float64)[:, None] * w[None]).sum(-1)[special]
        assert not np.isfinite(want).any()
        assert np.array_equal(np.isnan(y[special]), np.isnan(want))
        seen = ~np.isnan(want)
        assert np.array_equal(y[special][seen], want[seen])
        if not special.all():
            check_linear(y[~special], x[~special], w, big)


@pytest.mark.parametrize("dtype", [F16, BF16, E4M3])
def test_attention_over_q(dtype):
    """The output may be q itself: units split over CTAs, short ones, empty ones."""
    hq, hkv, d = 16, 2, 128
    for lens in ([20011], [4001, 0, 37, 1, 5099, 3777], [50] * 200):
        c = Cache(lens, 16, hkv, d, dtype, seed=len(lens))
        q = randn(len(lens), hq, d, seed=6)
        want = K.paged_attention(q, *c.args, c.lens, **c.scales)
        check_attention(c, q, want, None, d ** -0.5)
        ws = K.paged_attention_workspace(len(lens), hq, hkv, d, "cuda")
        for _ in range(10):
            over = q.clone()
            got = K.paged_attention(over, *c.args, c.lens, out=over, ws=ws, **c.scales)
            assert got is over and torch.equal(got, want)
    both = randn(3, hq, d, seed=7)
    with pytest.raises(_lib.MoEError, match="overlap"):
        K.paged_attention(both[:2], *Cache([9, 9], 16, hkv, d, dtype).args,
                          torch.tensor([9, 9], dtype=torch.int32).cuda(), out=both[1:],
                          **c.scales)


def test_broadcast_rows():
    """One bias for every row, one key and value for every token, one q for every
    sequence (strides of 0)."""
    rng = np.random.default_rng(8)
    raw, w, big = matrix(rng, 2, 100, 160)
    lw = K.LinearWeights(torch.from_numpy(raw.reshape(-1)).cuda(), 2, 100, 160)
    for T in (2, 9):
        x, bias = randn(T, 160, seed=T), randn(1, 100, seed=T + 1)
        y = K.linear(x, lw, residual=bias.expand(T, 100))
        check_linear(y.cpu().numpy(), x.cpu().numpy(), w, big, bias.cpu().numpy())
    hkv, d = 2, 64
    one, many = (Cache([9, 30, 17], 8, hkv, d, BF16, seed=9) for _ in range(2))
    q, kv, pos = randn(1, 4, d, seed=9), randn(1, hkv, d, seed=10), one.lens - 1
    freq = K.rope_inv_freq(d)
    turned = []
    for c, wide in ((one, lambda t: t.expand(3, -1, -1)), (many, lambda t: t.repeat(3, 1, 1))):
        turned.append(K.rope_append(wide(q), wide(kv), wide(kv), *c.args, pos, freq))
        turned.append(K.paged_attention(wide(q), *c.args, c.lens))
    assert torch.equal(turned[0], turned[2]) and torch.equal(turned[1], turned[3])
    assert torch.equal(one.k.view(torch.int16), many.k.view(torch.int16))
    assert torch.equal(one.v.view(torch.int16), many.v.view(torch.int16))


@pytest.mark.parametrize("dtype", [F16, BF16, E4M3])
@pytest.mark.parametrize("hq,hkv,d,window", [(12, 4, 64, 0), (8, 2, 128, 33), (6, 2, 256, 0)])
def test_equal_calls_whatever_ran_before(dtype, hq, hkv, d, window):
    """Slots that no row sees hold what earlier kernels left in shared memory; with
    and without a cap they count for nothing, not even in the last bit."""
    lens = [1, 20, 43, 7, 0, 65] * 40
    c = Cache(lens, 4, hkv, d, dtype, seed=d)
    q = 0.3 * randn(len(lens), hq, d, seed=d)
    ws = K.paged_attention_workspace(1, hq, hkv, d, "cuda")
    before = [Cache([200] * 150, 16, hkv, d, dtype, seed=1) for _ in range(2)]
    for t in (before[1].k, before[1].v):
        t.copy_(torch.full(t.shape, 3.0 if dtype == E4M3 else torch.inf, device="cuda").to(dtype))
    qb = 8 * randn(150, hq, d, seed=2)
    for cap in (0.0, 5.0, 30.0):
        want = None
        for b in before * 3:
            K.paged_attention(qb, *b.args, b.lens, ws=ws, **b.scales)
            got = K.paged_attention(q, *c.args, c.lens, window=window, softcap=cap, ws=ws,
                                    return_lse=True, **c.scales)
            if want is None:
                want = got
                check_attention(c, q, *got, d ** -0.5, window, cap)
            assert all(torch.equal(a, b) for a, b in zip(got, want)), cap

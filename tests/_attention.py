"""Plain 64-bit forms of the attention-half operators, their inputs and the
error bounds their tests hold them to."""
import math

import numpy as np
import torch

from linuxnightmaresuite_b200 import synth
from oracle import moe_oracle as orc

F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn
SCALES = {F16: (1.0, 1.0), BF16: (1.0, 1.0), E4M3: (0.03125, 0.0234375)}


class Cache:
    """A pool whose every slot is `fill` (NaN by default: a slot that nobody
    owns must not be read) and tables for sequences of the given lengths;
    entries behind a sequence's last page name no page."""

    def __init__(self, lens, page, hkv, d, dtype, layout="nhd", seed=0, fill=math.nan, spare=2,
                 width=None):
        g = torch.Generator().manual_seed(seed)
        need = [-(-max(n, 0) // page) for n in lens]
        total = sum(need) + spare
        shape = (total, page, hkv, d) if layout == "nhd" else (total, hkv, page, d)
        ks, vs = SCALES[dtype]
        self.k_scale, self.v_scale = ks, vs
        self.k = torch.full(shape, fill, dtype=torch.float32).to(dtype).cuda()
        self.v = torch.full(shape, fill, dtype=torch.float32).to(dtype).cuda()
        if layout != "nhd":
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        free = torch.randperm(total, generator=g).tolist()
        W = width or max(max(need), 1) + 1
        self.table = torch.full((len(lens), W), -7, dtype=torch.int32)
        for s, n in enumerate(need):
            for i in range(n):
                self.table[s, i] = free.pop()
        self.page = page
        # values of the owned slots, as the cache holds them (64 bits)
        self.kd, self.vd = [], []
        for s, n in enumerate(lens):
            n = max(n, 0)
            kv = torch.randn((2, n, hkv, d), generator=g)
            kv[0] /= ks
            kv[1] /= vs
            kv = kv.to(dtype).cuda()
            if n:
                pages, slots = self.where(s, range(n))
                if dtype == E4M3:
                    self.k.view(torch.uint8)[pages, slots] = kv[0].view(torch.uint8)
                    self.v.view(torch.uint8)[pages, slots] = kv[1].view(torch.uint8)
                else:
                    self.k[pages, slots], self.v[pages, slots] = kv[0], kv[1]
            self.kd.append(kv[0].double() * ks)
            self.vd.append(kv[1].double() * vs)
        self.table_d = self.table.cuda()
        self.lens = torch.tensor(lens, dtype=torch.int32).cuda()

    def where(self, s, positions):
        p = torch.tensor(list(positions))
        return self.table[s][p // self.page].long().cuda(), (p % self.page).cuda()

    @property
    def args(self):
        return self.k, self.v, self.table_d

    @property
    def scales(self):
        return dict(k_scale=self.k_scale, v_scale=self.v_scale)


def attend(q, kd, vd, scale, window=0, cap=0.0):
    """(out, lse, bound of |out - exact|, bound of |lse - exact|) of one
    sequence, 64 bits: q (hq, d), kd, vd (n, hkv, d).

    The bounds: a score is a sum of d products with q kept to 22 bits or more
    and f32 accumulation that may truncate, d / 16 <= 16 steps of 2^-23 of the
    sum of the products' magnitudes S: off by 2^-18 S at most with the
    scaling's roundings.  Its exponential carries that and 2^-20 of its own
    (argument and exp2 roundings, the probability's 22 bits); numerator and
    denominator each, so twice.  The sum over n keys is formed in f32 in parts
    of at least 16 keys: n / 16 roundings of 2^-24, and 2^-20 for the rest.
    A cap's tanh adds 2^-21 cap to a score."""
    hq, d = q.shape
    n, hkv, _ = kd.shape
    a = max(0, n - window) if window else 0
    kd, vd = kd[a:], vd[a:]
    if n == 0:
        return (torch.zeros_like(q), torch.full((hq,), -math.inf, dtype=torch.float64).to(q.device),
                torch.zeros_like(q), torch.zeros(hq, dtype=torch.float64, device=q.device))
    g = hq // hkv
    kr, vr = kd.repeat_interleave(g, 1), vd.repeat_interleave(g, 1)
    s = torch.einsum("hd,nhd->hn", q, kr) * scale
    S = (torch.einsum("hd,nhd->hn", q.abs(), kr.abs()) * abs(scale)).amax(-1)
    if cap:
        s = cap * torch.tanh(s / cap)
    p = torch.softmax(s, -1)
    out = torch.einsum("hn,nhd->hd", p, vr)
    ds = S * 2.0 ** -18 + cap * 2.0 ** -21
    vmax = vr.abs().amax((0, 2))
    tol = vmax * (2 * (ds + 2.0 ** -20) + (n / 16) * 2.0 ** -24 + 2.0 ** -20)
    lse = torch.logsumexp(s, -1)
    return out, lse, tol[:, None].expand(hq, d), ds + 2.0 ** -19 + lse.abs() * 2.0 ** -22


def check_attention(c, q, out, lse, scale, window=0, cap=0.0):
    for s in range(q.shape[0]):
        o, l, to, tl = attend(q[s].double(), c.kd[s], c.vd[s], scale, window, cap)
        assert (out[s].double() - o).abs().le(to).all(), (
            s, (out[s].double() - o).abs().max().item(), to.max().item())
        if lse is not None:
            if c.kd[s].shape[0] == 0:
                assert torch.isneginf(lse[s]).all()
            else:
                assert (lse[s].double() - l).abs().le(tl).all(), (s, lse[s], l)


def rotate(x, positions, inv_freq, interleaved):
    """x (T, H, d) f64 turned by its positions, and the bound of an f32 form:
    sin and cos within 2^-22 (two ulp and the angle's remainder), two products
    and one sum of 2^-24 each: 2^-21 (|x1| + |x2|)."""
    rot = 2 * inv_freq.numel()
    a = positions.double()[:, None, None] * inv_freq
    c, s = a.cos(), a.sin()
    y, bound = x.clone(), torch.zeros_like(x)
    i = torch.arange(rot // 2, device=x.device)
    e0, e1 = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    x0, x1 = x[..., e0], x[..., e1]
    y[..., e0], y[..., e1] = x0 * c - x1 * s, x1 * c + x0 * s
    bound[..., e0] = bound[..., e1] = (x0.abs() + x1.abs()) * 2.0 ** -21
    return y, bound


def check_stored(stored, value, bound, dtype, scale):
    """A cache entry is value / scale, off by the bound of the value and half
    a step of the type (half of its smallest step below the normal range)."""
    tiny = {F16: 2.0 ** -25, BF16: 0.0, E4M3: 2.0 ** -10}[dtype]
    want = value / scale
    if dtype == E4M3:
        want = want.clamp(-448, 448)
    tol = bound / scale + (want.abs() + bound / scale) * (torch.finfo(dtype).eps / 2) + tiny
    assert ((stored.double() - want).abs() <= tol * (1 + 2.0 ** -20)).all()


def matrix(rng, qtype, rows, cols, scale=0.01):
    """(raw block bytes, 64-bit values, |d| (|q| + offset) of each weight)."""
    raw = synth.quant_matrix(rng, qtype, 1, rows, cols, scale)
    w = orc.dequantize_matrix(raw.reshape(-1), qtype, rows, cols).astype(np.float64)
    b = raw.reshape(rows, cols // 32, -1)
    d = np.abs(b[..., :2].copy().view(np.float16).astype(np.float64))
    big = np.abs(w) + np.repeat(d, 32, axis=-1).reshape(rows, cols) * (8 if qtype == 2 else 128)
    return raw, w, big


def check_linear(y, x, w, big, residual=None):
    """y = x w^T.  x is kept to 22 bits or more (2^-22), a block of 32 products
    and its offset correction is summed with two truncations of 2^-23 each of
    the magnitudes met, and the cols / 32 blocks with roundings of 2^-24; x
    parts far below the row's largest are kept to 2^-39 of that."""
    x = x.astype(np.float64)
    ref = x @ w.T
    mag = np.abs(x) @ big.T + 2.0 ** -17 * np.abs(x).max(1, keepdims=True) * big.sum(1)
    tol = mag * (2.0 ** -21 + (w.shape[1] / 32) * 2.0 ** -24)
    if residual is not None:
        ref = ref + residual
        tol = tol + np.abs(ref) * 2.0 ** -23
    err = np.abs(y.astype(np.float64) - ref)
    assert (err <= tol).all(), (err.max(), (err / tol).max())

"""Bounds of the norm of an operator's error, next to the bounds of single
elements: independent roundings add up like the root of a sum of squares, so a
norm shows a rounding, a key or a tile that is lost where the worst case of a
single element of a long sum hides it."""
import numpy as np
import torch


def attention_errors(q, kd, vd, out, lse, scale, window=0, cap=0.0):
    """(|out - exact| / bound of each head's norm, |lse - exact| / bound) of one
    sequence, 64 bits: q (hq, d), kd, vd (n, hkv, d).

    A score s_j is off by roundings of its products, which are independent: q in
    22 bits or more, at most 16 accumulation steps that truncate, in units of
    the products' root of squares S: 2^-19 S; and by roundings of itself (scale,
    cap, argument of the exponential): 2^-21 |s|.  An exponential, its two parts
    and eight accumulation steps add 2^-19.  So each p_j v_j is off by at most
    E = 2^-19 (1 + S) + 2^-21 |s|, independently, and their sum by E times the
    root of the sum of |p_j v_j|^2.  The sum that divides is common to all:
    2^-20 of the output."""
    hq, d = q.shape
    n, hkv, _ = kd.shape
    a = max(0, n - window) if window else 0
    g = hq // hkv
    k, v = kd[a:].repeat_interleave(g, 1), vd[a:].repeat_interleave(g, 1)
    s = torch.einsum("hd,nhd->hn", q, k) * scale
    S = torch.einsum("hd,nhd->hn", q ** 2, k ** 2).amax(-1).sqrt() * abs(scale)
    if cap:
        s = cap * torch.tanh(s / cap)
    p = torch.softmax(s, -1)
    exact = torch.einsum("hn,nhd->hd", p, v)
    E = 2.0 ** -19 * (1 + S) + 2.0 ** -21 * s.abs().amax(-1)
    R = ((p * v.norm(dim=-1).T) ** 2).sum(-1).sqrt()
    err = (out - exact).norm(dim=-1) / (E * R + 2.0 ** -20 * exact.norm(dim=-1))
    if lse is None:
        return err, torch.zeros_like(err)
    l = torch.logsumexp(s, -1)
    return err, (lse - l).abs() / (E + 2.0 ** -20 + l.abs() * 2.0 ** -22)


def check_attention_norms(c, q, out, lse, scale, window=0, cap=0.0):
    for s in range(q.shape[0]):
        if c.kd[s].shape[0]:
            eo, el = attention_errors(q[s].double(), c.kd[s], c.vd[s], out[s].double(),
                                      lse[s].double(), scale, window, cap)
            assert (eo <= 1).all() and (el <= 1).all(), (s, eo.max().item(), el.max().item())


def linear_errors(y, x, w, residual=None):
    """|y - exact| / bound of each row's norm, y = x w^T.  Each product carries x
    in 22 bits or more and its share of two truncating accumulation steps of a
    block of 32, 2^-20 together; the cols / 32 blocks are added in f32, each sum
    off by 2^-24 of what is there at most, independently.  Both count against the
    root of the sum of the products' squares; the last additions are off by 2^-23
    of the result."""
    x = x.astype(np.float64)
    exact = x @ w.T
    R = np.sqrt((x ** 2 @ (w ** 2).sum(0)))
    if residual is not None:
        exact = exact + residual
    bound = (2.0 ** -20 + 2.0 ** -24 * (w.shape[1] / 32) ** 0.5) * R
    err = np.linalg.norm(y.astype(np.float64) - exact, axis=1)
    return err / (bound + 2.0 ** -23 * np.linalg.norm(exact, axis=1))

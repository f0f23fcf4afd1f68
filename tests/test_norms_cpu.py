"""The norm bounds let the operators' own roundings pass and nothing coarser:
one part of a probability or of x, a key or a tile that is lost, met twice or
paired with another's values."""
import numpy as np
import pytest
import torch

from ._attention import matrix
from ._norms import attention_errors, linear_errors

LINEAR_SIZES = [(203, 1056), (96, 8192), (64, 32768), (40, 65536), (300, 512)]


def parts(x, dtype, n):
    """x kept as the sum of n parts of a 16-bit type."""
    y = torch.zeros_like(x)
    for _ in range(n):
        y = y + (x - y).float().to(dtype).double()
    return y


def inputs(n, d, seed, size):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(s, generator=g).double() for s in ((2, d), (n, 1, d), (n, 1, d)))
    return q * size, k, v


def attend(q, k, v, p_parts=None, q_parts=None):
    """Attention with q (scaled by its largest) and the probabilities in parts."""
    if q_parts:
        top = 2.0 ** (10 - torch.floor(torch.log2(q.abs().amax(-1, keepdim=True))))
        q = parts(q * top, *q_parts) / top
    s = torch.einsum("hd,nd->hn", q, k[:, 0]) * q.shape[1] ** -0.5
    p = torch.exp2((s - s.amax(-1, keepdim=True)) / np.log(2) + 7)
    l = p.sum(-1, keepdim=True)
    if p_parts:
        p = parts(p, *p_parts)
    return p @ v[:, 0] / l


def worst(q, k, v, out):
    return attention_errors(q, k, v, out.float().double(), None, q.shape[1] ** -0.5)[0].max()


@pytest.mark.parametrize("n,d,size", [(1, 64, 1.5), (17, 128, 1.5), (777, 64, 1.5),
                                      (40001, 128, 0.3), (30011, 256, 0.3)])
def test_attention_norms_tell_roundings_apart(n, d, size):
    q, k, v = inputs(n, d, n, size)
    assert worst(q, k, v, attend(q, k, v, (torch.float16, 2), (torch.float16, 2))) < 0.5
    assert worst(q, k, v, attend(q, k, v, (torch.bfloat16, 3), (torch.bfloat16, 3))) < 0.5
    if n > 1:                                       # one key: p is a power of two, q counts for nothing
        for t in (torch.float16, torch.bfloat16):
            assert worst(q, k, v, attend(q, k, v, p_parts=(t, 1))) > 4
            assert worst(q, k, v, attend(q, k, v, q_parts=(t, 1))) > 4


@pytest.mark.parametrize("n,d", [(777, 64), (40001, 128), (30011, 256)])
def test_attention_norms_miss_no_tile(n, d):
    q, k, v = inputs(n, d, n, 0.3)
    s = torch.einsum("hd,nd->hn", q, k[:, 0]) * d ** -0.5
    p = torch.softmax(s, -1)
    out = p @ v[:, 0]
    tiles = torch.randperm(n // 32, generator=torch.Generator().manual_seed(1))[:20].tolist()
    for a, b in zip(tiles, tiles[1:]):
        a, b = slice(32 * a, 32 * a + 32), slice(32 * b, 32 * b + 32)
        part = p[:, a] @ v[a, 0]
        one = p[:, a.start:a.start + 1] * v[a.start]
        for wrong in (out - part, out + part,                                # values lost, twice
                      (out - part) / (1 - p[:, a].sum(-1, keepdim=True)),    # the tile, with its sum
                      out - one, (out - one) / (1 - p[:, a.start:a.start + 1]),   # one key
                      out - part - p[:, b] @ v[b, 0] + p[:, a] @ v[b, 0] + p[:, b] @ v[a, 0]):
            assert worst(q, k, v, wrong) > 10


@pytest.mark.parametrize("qtype", [2, 8])
@pytest.mark.parametrize("rows,cols", LINEAR_SIZES)
def test_linear_norms_tell_roundings_apart(qtype, rows, cols):
    rng = np.random.default_rng(cols)
    _, w, _ = matrix(rng, qtype, rows, cols)
    x = rng.standard_normal((2, cols), dtype=np.float32)
    top = 2.0 ** (14 - np.floor(np.log2(np.abs(x).max(1, keepdims=True))))
    xs = torch.from_numpy(x).double() * torch.from_numpy(top).double()
    for n, passes in ((2, True), (1, False)):
        kept = (parts(xs, torch.float16, n) / torch.from_numpy(top).double()).numpy()
        err = linear_errors((kept @ w.T).astype(np.float32), x, w)
        assert (err < 0.5).all() if passes else (err > 10).all()
    res = rng.standard_normal((2, rows), dtype=np.float32)
    assert (linear_errors((x @ w.T + res).astype(np.float32), x, w, res) < 0.5).all()
    lost = x.copy()
    lost[:, 64:128] = 0                             # a tile of columns
    assert (linear_errors(lost @ w.T, x, w) > 100).all()

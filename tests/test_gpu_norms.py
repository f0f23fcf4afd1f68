"""Attention and linear against 64-bit forms by the norm of the error, at the
shapes where single elements' bounds are wide: long sequences that are split,
rows of many thousand columns."""
import numpy as np
import pytest
import torch

from linuxnightmaresuite_b200 import kernels as K

from ._attention import BF16, E4M3, F16, Cache, matrix
from ._norms import check_attention_norms, linear_errors
from .test_gpu_attention import randn

pytestmark = pytest.mark.gpu

RAGGED = [1, 15, 16, 17, 0, 63, 64, 65, 129, 777, 31]


@pytest.mark.parametrize("dtype", [F16, BF16, E4M3])
@pytest.mark.parametrize("hq,hkv,d,page,lens,window,cap,size", [
    (8, 2, 128, 16, RAGGED, 0, 0.0, 1.5),
    (16, 16, 64, 24, RAGGED, 0, 0.0, 1.5),
    (4, 1, 256, 7, RAGGED, 0, 0.0, 1.5),
    (10, 2, 80, 1, RAGGED, 0, 0.0, 1.5),      # five heads share one
    (16, 1, 64, 16, [20000, 9, 12345], 0, 0.0, 0.3),
    (8, 2, 128, 16, [40001], 0, 0.0, 0.3),
    (4, 4, 256, 16, [30011, 5000], 0, 0.0, 0.3),
    (6, 2, 128, 16, [99, 1500, 400], 100, 30.0, 2.0),
    (8, 2, 128, 32, [600, 90], 0, 0.0, 60.0),   # scores in the hundreds
])
def test_attention_norms(dtype, hq, hkv, d, page, lens, window, cap, size):
    c = Cache(lens, page, hkv, d, dtype, seed=d + page)
    q = size * randn(len(lens), hq, d, seed=hq)
    out, lse = K.paged_attention(q, *c.args, c.lens, window=window, softcap=cap, return_lse=True,
                                 **c.scales)
    check_attention_norms(c, q, out, lse, d ** -0.5, window, cap)


@pytest.mark.parametrize("qtype,rows,cols,tokens", [(q, *shape) for q in (2, 8) for shape in (
    (203, 1056, (1, 2, 3, 4, 5, 8, 16, 17)),
    (4096, 8192, (1, 2, 4, 8, 16)),
    (64, 32768, (1, 3, 16)),
    (65541, 512, (1, 13)),
)] + [(2, 40, 65536, (1, 2, 7))])               # Q8_0 this wide does not fit
def test_linear_norms(qtype, rows, cols, tokens):
    rng = np.random.default_rng(rows)
    raw, w, _ = matrix(rng, qtype, rows, cols)
    lw = K.LinearWeights(torch.from_numpy(raw.reshape(-1)).cuda(), qtype, rows, cols)
    for T in tokens:
        x = rng.standard_normal((T, cols), dtype=np.float32)
        res = rng.standard_normal((T, rows), dtype=np.float32) if T % 2 else None
        y = K.linear(torch.from_numpy(x).cuda(), lw,
                     residual=None if res is None else torch.from_numpy(res).cuda())
        err = linear_errors(y.cpu().numpy(), x, w, res)
        assert (err <= 1).all(), (T, err.max())

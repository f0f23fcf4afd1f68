"""Decode steps captured at several batch sizes and replayed in turn, with
other sizes called and memory taken in between."""
import gc
import math

import pytest
import torch

from linuxnightmaresuite_b200.attention import PagedKVCache

from ._attention import F16
from .test_gpu_attention import _decoder, randn

pytestmark = pytest.mark.gpu

SIZES = (2, 3, 5)


def _caches(layers, seqs):
    cs = [PagedKVCache(64, 8, 2, 64, seqs, 8, F16) for _ in range(layers)]
    for c in cs:
        for s in range(seqs):
            c.reserve(s, 60)
    return cs


def _others(fill):
    """Tensors of many sizes in whatever memory is free."""
    gc.collect()
    return [torch.full((1 << k,), fill, device="cuda") for k in range(6, 22) for _ in range(4)]


def _two_sizes(step, eager, caches, alone):
    """Captures step(x, out, caches, positions, lens) at each size, calls a larger
    one, and replays all in turn against `eager` on caches of its own."""
    graphs = {}
    for T in SIZES:
        x, out = randn(T, 512, seed=T), torch.empty((T, 512), device="cuda")
        pos = torch.zeros(T, dtype=torch.int32, device="cuda")
        lens = pos + 1
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(x, out, caches, pos, lens)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(x, out, caches, pos, lens)
        graphs[T] = (g, x, out, pos, lens)
    big = max(SIZES) + 3
    step(randn(big, 512), torch.empty((big, 512), device="cuda"), caches,
         torch.full((big,), -1, dtype=torch.int32, device="cuda"),
         torch.zeros(big, dtype=torch.int32, device="cuda"))
    for at in range(20):
        others = _others(math.nan if at % 2 else 1.0)
        for T, (g, x, out, pos, lens) in graphs.items():
            x.copy_(randn(T, 512, seed=100 * T + at))
            pos.fill_(at)
            lens.fill_(at + 1)
            out.fill_(math.nan)
            g.replay()
            want = torch.empty_like(out)
            eager(x, want, alone, pos, lens)
            assert torch.equal(out, want), (at, T)
        for t in others:                            # nothing wrote outside its buffers
            assert torch.isnan(t).all() if at % 2 else (t == 1.0).all()
        del others


def test_attention_layer_two_sizes_captured():
    one, two = (_decoder(F16, 2, layers=1)[0].attention[0] for _ in range(2))

    def run(layer):
        return lambda x, out, c, pos, lens: layer.forward(x, c[0], pos, lens, residual=x, out=out)
    _two_sizes(run(one), run(two), _caches(1, 8), _caches(1, 8))
    assert one.device_status() == 0 and two.device_status() == 0


def _step(stack):
    return lambda x, out, c, pos, lens: stack.forward(x, out=out, caches=c, positions=pos,
                                                      seq_lens=lens)


def test_decoder_two_sizes_captured():
    one, two = (_decoder(F16, 2)[0] for _ in range(2))
    _two_sizes(_step(one), _step(two), _caches(2, 8), _caches(2, 8))
    for layer in one.attention + two.attention + one.layers + two.layers:
        assert layer.device_status() == 0


def test_first_call_captured():
    """Layers whose first call is captured: what the graph's replays clear is not
    there for calls before the first of them."""
    warm, stack = (_decoder(F16, 2)[0] for _ in range(2))
    caches, alone = _caches(2, 3), _caches(2, 3)
    x, out = randn(3, 512, seed=1), torch.empty((3, 512), device="cuda")
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")
    lens = pos + 1
    want = torch.empty_like(out)
    _step(warm)(x, want, alone, pos, lens)          # what the library loads at its first calls
    others = _others(math.nan)
    del others
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        _step(stack)(x, out, caches, pos, lens)
    eager = torch.empty_like(out)
    _step(stack)(x, eager, caches, pos, lens)
    assert torch.equal(eager, want)
    assert all(layer.device_status() == 0 for layer in stack.attention)
    for _ in range(3):
        out.fill_(math.nan)
        g.replay()
        assert torch.equal(out, want)
    assert all(layer.device_status() == 0 for layer in stack.layers)

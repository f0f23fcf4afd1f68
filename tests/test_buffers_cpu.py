"""Buffers that a captured CUDA graph may hold keep their address and their
memory, whatever sizes are called in between."""
import gc
import types
import weakref

import pytest
import torch

from linuxnightmaresuite_b200 import build, kernels as K
from linuxnightmaresuite_b200.attention import AttentionLayer
from linuxnightmaresuite_b200.moe_forward import MoELayer
from linuxnightmaresuite_b200.stacked import StackedEP, StackedMoE


def _attention(hq=4, hk=2, d=64, dim=128):
    build.build()
    cpu = torch.device("cpu")
    qkv = types.SimpleNamespace(rows=(hq + 2 * hk) * d, cols=dim, device=cpu)
    return AttentionLayer(qkv, types.SimpleNamespace(rows=dim, cols=hq * d, device=cpu), hq, hk, d)


def test_attention_buffers_of_a_size_stay():
    layer = _attention()
    held, at = [], {}
    for T in (2, 3, 2, 1, 64, 7, 2, 3, 1, 0):
        parts = layer._buffers(T)
        where = [t.data_ptr() for t in parts]
        assert at.setdefault(T, where) == where
        assert parts[0].shape == (T, 8 * 64) and parts[1].shape == (T, 4, 64)
        held += [weakref.ref(t.untyped_storage()) for t in parts]
        del parts
    gc.collect()
    assert all(r() is not None for r in held)


def test_attention_has_one_workspace():
    """Its counters are zero before the first call, also where that is captured,
    and one status word gathers what calls of every size report."""
    layer = _attention()
    a, b = layer._buffers(2)[2], layer._buffers(3)[2]
    assert a.data_ptr() == b.data_ptr() and a.numel() == b.numel()
    assert not a.any()


class _Step:
    """Stands for a layer on the host; notes the rows that it is given."""

    def __init__(self, seen):
        self.seen = seen

    def forward_batch(self, xn, residual=None, out=None):
        self.seen.append(xn)

    def forward(self, xn, out=None, residual=None):
        self.seen.append(xn)


@pytest.mark.parametrize("kind", [StackedMoE, StackedEP])
def test_stacked_buffer_of_a_size_stays(kind, monkeypatch):
    monkeypatch.setattr(K, "rms_norm", lambda x, w, eps, out: out)
    seen, at, held = [], {}, []
    stack = kind([_Step(seen)], [None])
    for T in (2, 3, 2, 1, 64, 7, 2, 3, 1):
        x = torch.zeros(T, 32)
        stack.forward(x)
        xn = seen.pop()
        assert xn.shape == x.shape
        assert at.setdefault(T, xn.data_ptr()) == xn.data_ptr()
        held.append(weakref.ref(xn.untyped_storage()))
        del xn
    gc.collect()
    assert all(r() is not None for r in held)


def _moe(monkeypatch):
    status = {}                                     # by address, as the device would set it
    layer = MoELayer.__new__(MoELayer)
    layer.router = types.SimpleNamespace(device=torch.device("cpu"))
    layer._ws, layer._held = None, []
    layer.weights = types.SimpleNamespace(workspace_bytes=lambda T: 256 + 100 * T)
    monkeypatch.setattr(K, "read_status", lambda ws: status.pop(ws.data_ptr(), 0))
    return layer, status


def test_moe_workspace_that_a_graph_may_hold_stays(monkeypatch):
    """A larger batch brings a larger workspace; the one before is kept, and what
    a replayed graph reports into it is read."""
    layer, status = _moe(monkeypatch)
    assert layer.device_status() == 0
    held, total = [], 0
    for T in list(range(1, 200)) + [5, 1]:
        ws = layer._workspace(T)
        assert ws.numel() >= 256 + 100 * T and ws.dtype == torch.uint8 and not ws[:256].any()
        if not any(r() is ws.untyped_storage() for r in held):
            held.append(weakref.ref(ws.untyped_storage()))
            total += ws.numel()
        first = ws if T == 1 and len(held) == 1 else first
        last = ws
        del ws
    gc.collect()
    assert all(r() is not None for r in held)
    assert last.numel() >= 256 + 100 * 199 and total <= 4 * last.numel()   # growth by halves
    status[first.data_ptr()] = 1
    status[last.data_ptr()] = 4
    assert layer.device_status() == 5
    assert layer.device_status() == 0

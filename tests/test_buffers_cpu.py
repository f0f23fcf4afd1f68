"""Buffers that a captured CUDA graph may hold keep their address and their
memory, whatever sizes are called in between."""
import gc
import types
import weakref

import torch

from linuxnightmaresuite_b200 import build
from linuxnightmaresuite_b200.attention import AttentionLayer


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

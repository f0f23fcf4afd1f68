"""Host side of shared prefixes and shrinking caches: refusals of the C entries before
any device work, the ctypes mirrors, the page bookkeeping."""
import ctypes
import math

import pytest
import torch

from linuxnightmaresuite_b200 import _lib, attention, kernels as K
from linuxnightmaresuite_b200.attention import PagedKVCache
from linuxnightmaresuite_b200.stacked import StackedMoE

from .test_attention_cpu import BAD_CACHES, cache, lib, test_argument_record_matches_header as _match

F = 1 << 20                            # aligned addresses that no refused call follows


def norm_append(c, mass=0, held=0, slots=0, width=0, eps=1e-6, T=2, rot=64, q=F):
    return _lib.MoENormAppendArgs(
        append=_lib.MoERopeAppendArgs(
            cache=c, q=q, k=F, v=F, q_tok_stride=256, q_head_stride=64, k_tok_stride=128,
            k_head_stride=64, v_tok_stride=128, v_head_stride=64, positions=F, inv_freq=F,
            q_out=2 * F, qo_tok_stride=256, qo_head_stride=64, T=T, q_heads=4, rot=rot),
        q_norm=F, k_norm=F, slots=slots, mass=mass, held=held, ledger_slots=width, eps=eps)


def mass(c, q=F, lse=F, mass=F, out=F, width=64, hq=4, lens=F, max_len=0, window=0, scale=0.1, cap=0.0):
    return _lib.MoEAttentionMassArgs(
        cache=c, q=q, q_seq_stride=256, q_head_stride=64, seq_lens=lens, lse=lse, mass=mass, out=out,
        ledger_slots=width, q_heads=hq, max_len=max_len, window=window, scale=scale, softcap=cap)


def evict(c, lens=F, mass=F, held=2 * F, mass_out=F, held_out=2 * F, lens_out=F, width=64, wide=64,
          keep=32, recent=4, max_len=0):
    return _lib.MoECacheEvictArgs(
        cache=c, seq_lens=lens, mass=mass, held=held, mass_out=mass_out, held_out=held_out,
        lens_out=lens_out, ledger_slots=width, out_slots=wide, keep=keep, recent=recent,
        max_len=max_len)


def prefix(c, pages=2, form=0, list_=F, q=F, out=4 * F, ws=8 * F, nbytes=1 << 30, hq=4, window=0,
           scale=0.1, cap=0.0, max_len=0, lens=F):
    return _lib.MoEPrefixAttentionArgs(
        attention=_lib.MoEPagedAttentionArgs(
            cache=c, q=q, q_seq_stride=256, q_head_stride=64, seq_lens=lens, out=out, lse=0,
            workspace=ws, workspace_bytes=nbytes, q_heads=hq, max_len=max_len, window=window,
            scale=scale, softcap=cap),
        prefix=list_, prefix_pages=pages, form=form)


CALLS = {"moe_norm_append_record": norm_append, "moe_attention_mass_record": mass,
         "moe_cache_evict_record": evict, "moe_prefix_attention_record": prefix}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("change,status,words", BAD_CACHES)
def test_bad_caches_are_refused(lib, name, change, status, words):
    a = CALLS[name](cache(**change))
    assert getattr(lib, name)(ctypes.byref(a)) == getattr(_lib, "MOE_ERR_" + status)
    assert words in _lib.last_error()
    assert getattr(lib, name)(None) == _lib.MOE_ERR_INVALID


def refused(lib, name, status="INVALID", words=None, **kw):
    a = CALLS[name](cache(), **kw)
    assert getattr(lib, name)(ctypes.byref(a)) == getattr(_lib, "MOE_ERR_" + status), kw
    assert words is None or words in _lib.last_error(), (kw, _lib.last_error())


def test_bad_norm_append_arguments_are_refused(lib):
    for kw in (dict(T=-1), dict(rot=63), dict(rot=66), dict(q=0), dict(eps=-1.0), dict(eps=math.nan),
               dict(mass=F), dict(held=F), dict(mass=F, held=F), dict(mass=F, held=F, width=-3),
               dict(T=5)):
        refused(lib, "moe_norm_append_record", **kw)
    a = norm_append(cache(), T=0)
    assert lib.moe_norm_append_record(ctypes.byref(a)) == _lib.MOE_OK


def test_bad_mass_arguments_are_refused(lib):
    n = "moe_attention_mass_record"
    for kw in (dict(hq=0), dict(hq=3), dict(max_len=-1), dict(window=-1), dict(scale=math.inf),
               dict(cap=-1.0), dict(width=0), dict(q=0), dict(lse=0), dict(mass=0), dict(out=0),
               dict(lens=0)):
        refused(lib, n, **kw)
    ledger = 4 * 2 * 64 * 4                         # bytes
    for off in (4, -4, ledger - 4, 4 - ledger):
        refused(lib, n, words="overlap", out=F + off)
    a = mass(cache(seqs=0), q=0)
    assert lib.moe_attention_mass_record(ctypes.byref(a)) == _lib.MOE_OK


def test_bad_evict_arguments_are_refused(lib):
    n = "moe_cache_evict_record"
    for kw in (dict(keep=0), dict(keep=-1), dict(recent=-1), dict(recent=33), dict(max_len=-1),
               dict(width=0), dict(wide=0), dict(lens=0), dict(mass=0), dict(held=0),
               dict(mass_out=0), dict(held_out=0), dict(lens_out=0)):
        refused(lib, n, **kw)
    refused(lib, n, words="ledgers of the result", wide=31, mass_out=4 * F, held_out=5 * F)
    ledger = 4 * 2 * 64 * 4
    for kw in (dict(mass_out=F + 4), dict(mass_out=F - 4), dict(held_out=2 * F + ledger - 4),
               dict(held_out=F), dict(mass_out=2 * F), dict(mass=2 * F, mass_out=2 * F),
               dict(mass_out=F, wide=40, held_out=4 * F), dict(lens_out=F + 4)):
        refused(lib, n, words="overlap", **kw)
    # rows of a cache that share memory can not be moved
    for kw in (dict(page_stride=0), dict(head_stride=0), dict(head_stride=56)):
        a = evict(cache(**kw))
        assert lib.moe_cache_evict_record(ctypes.byref(a)) == _lib.MOE_ERR_INVALID
        assert "share memory" in _lib.last_error()
    a = evict(cache(table_width=1 << 20, table_stride=1 << 20), width=1 << 24, wide=1 << 24,
              held=1 << 40, held_out=1 << 40)
    assert lib.moe_cache_evict_record(ctypes.byref(a)) == _lib.MOE_ERR_UNSUPPORTED
    assert "163840" in _lib.last_error()
    a = evict(cache(seqs=0), lens=0)
    assert lib.moe_cache_evict_record(ctypes.byref(a)) == _lib.MOE_OK


def test_bad_prefix_arguments_are_refused(lib):
    n = "moe_prefix_attention_record"
    for kw in (dict(hq=0), dict(hq=3), dict(max_len=-1), dict(scale=math.nan), dict(cap=-1.0),
               dict(q=0), dict(out=0), dict(ws=0), dict(lens=0), dict(list_=0), dict(pages=-1),
               dict(pages=9), dict(form=3), dict(form=-1), dict(ws=8 * F + 8), dict(out=4 * F + 4),
               dict(window=-1), dict(out=F + 4)):
        refused(lib, n, **kw)
    refused(lib, n, "UNSUPPORTED", "window", window=5)
    refused(lib, n, "WORKSPACE", nbytes=1 << 16)
    a = prefix(cache(seqs=0), q=0)
    assert lib.moe_prefix_attention_record(ctypes.byref(a)) == _lib.MOE_OK
    size = ctypes.c_size_t()
    assert lib.moe_prefix_attention_workspace_bytes(4, 4, 2, 64, ctypes.byref(size)) == _lib.MOE_OK
    small = size.value
    assert lib.moe_prefix_attention_workspace_bytes(4000, 4, 2, 64, ctypes.byref(size)) == _lib.MOE_OK
    assert size.value > small
    for heads in ((1, 1, 64), (8, 2, 128), (16, 4, 256), (24, 1, 96)):
        last = 0                                    # a workspace serves fewer sequences too
        for seqs in range(1, 1500, 7):
            assert lib.moe_prefix_attention_workspace_bytes(seqs, *heads, ctypes.byref(size)) == 0
            assert size.value >= last, (heads, seqs)
            last = size.value
    for bad in ((-1, 4, 2, 64), (4, 5, 2, 64), (4, 4, 0, 64), (4, 4, 2, 257)):
        assert lib.moe_prefix_attention_workspace_bytes(*bad, ctypes.byref(size)) == \
            _lib.MOE_ERR_INVALID


@pytest.mark.parametrize("name, mirror", [
    ("moe_attention_mass_args", _lib.MoEAttentionMassArgs),
    ("moe_cache_evict_args", _lib.MoECacheEvictArgs)])
def test_argument_record_matches_header(name, mirror):
    _match(name, mirror)


def test_nested_records_have_the_size_of_their_parts():
    assert ctypes.sizeof(_lib.MoEPrefixAttentionArgs) == \
        ctypes.sizeof(_lib.MoEPagedAttentionArgs) + 16
    assert ctypes.sizeof(_lib.MoENormAppendArgs) == ctypes.sizeof(_lib.MoERopeAppendArgs) + 56


def test_wrappers_refuse_host_tensors():
    k = torch.zeros((2, 4, 1, 64), dtype=torch.float16)
    t = torch.zeros((1, 2), dtype=torch.int32)
    q, m = torch.zeros(1, 2, 64), torch.zeros(1, 1, 8)
    for call in (lambda: K.prefix_attention(q, k, k, t, t[0, :1], t[0]),
                 lambda: K.attention_mass(q, k, t, t[0, :1], q[..., 0], m),
                 lambda: K.cache_evict(k, k, t, t[0, :1], m, m.int(), 4)):
        with pytest.raises(TypeError, match="CUDA"):
            call()


def test_pages_are_shared_and_trimmed():
    c = PagedKVCache(10, 4, 2, 16, max_seqs=4, max_pages_per_seq=6, device="cpu")
    c.reserve(0, 14)                                # four pages
    c.share(1, 0, 12)
    c.share(2, 1, 8)
    assert c.free_pages == 6
    assert torch.equal(c.block_table[1, :3], c.block_table[0, :3]) and c.block_table[1, 3] == -1
    assert torch.equal(c.prefix(2, 8), c.block_table[0, :2])
    c.reserve(1, 13)                                # a page of its own behind them
    assert c.free_pages == 5 and c.block_table[1, 3] != c.block_table[0, 3]
    for bad in (lambda: c.share(1, 0, 4), lambda: c.share(3, 0, 6), lambda: c.share(3, 2, 12),
                lambda: c.share(3, 0, -4), lambda: c.prefix(0, 7), lambda: c.prefix(0, 28)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: c.share(4, 0, 4), lambda: c.share(3, -1, 4), lambda: c.prefix(9, 4),
                lambda: c.trim(4, 0)):
        with pytest.raises(IndexError):
            bad()
    c.release(0)                                    # three pages are still in use
    assert c.free_pages == 6 and (c.block_table[0] == -1).all()
    c.trim(1, 9)
    assert c.free_pages == 7 and c.block_table[1].tolist()[3:] == [-1] * 3
    c.trim(1, 100)
    c.trim(1, 4)                                    # two of the pages are sequence 2's too
    assert c.free_pages == 8
    c.release(2)
    assert c.free_pages == 9
    c.release(1)
    c.release(1)
    assert c.free_pages == 10 and sorted(c._free) == list(range(10)) and not any(c._users)
    c.share(3, 0, 0)
    assert c.prefix(3, 0).numel() == 0


def test_ledger_of_a_cache():
    c = PagedKVCache(6, 4, 2, 16, max_seqs=3, max_pages_per_seq=4, device="cpu", track=True)
    assert c.mass.shape == c.held.shape == (3, 2, 16)
    c.reserve(0, 8)
    with pytest.raises(ValueError, match="shares no pages"):
        c.share(1, 0, 4)
    plain = PagedKVCache(6, 4, 2, 16, max_seqs=3, device="cpu")
    t = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="ledger"):
        plain.evict(t, 4)
    with pytest.raises(ValueError, match="ledger"):
        plain.weigh(torch.zeros(3, 2, 16), t, torch.zeros(3, 2))
    with pytest.raises(ValueError, match="window"):
        plain.attend(torch.zeros(3, 2, 16), t, window=3, prefix=t)
    assert attention.evict([], t, 4) is t


def test_a_prefix_outlives_the_sequence_that_it_came_from():
    c = PagedKVCache(10, 4, 2, 16, max_seqs=4, max_pages_per_seq=6, device="cpu")
    c.reserve(0, 14)
    c.share(1, 0, 8)
    pages = c.prefix(0, 8)
    first = pages.tolist()
    assert first == c.block_table[0, :2].tolist()
    assert c.prefix(1, 8) is pages                  # the same list, made once
    c.release(0)
    c.reserve(0, 24)                                # another prompt in its place
    assert pages.tolist() == first == c.block_table[1, :2].tolist()
    assert c.prefix(0, 8).tolist() == c.block_table[0, :2].tolist() != first
    assert c.prefix(1, 8) is pages
    # pages that went back and came again belong to another list
    c.release(1)
    c.release(0)
    c.reserve(2, 4)
    c.share(3, 2, 4)
    c.trim(2, 0)
    c.reserve(2, 24)
    for s in (2, 3):
        for n in range(len(c._held[s]) + 1):
            assert c.prefix(s, 4 * n).tolist() == c._held[s][:n] == c.block_table[s, :n].tolist()
    c.trim(2, 8)
    c.reserve(2, 16)
    for n in range(5):
        assert c.prefix(2, 4 * n).tolist() == c._held[2][:n]
    with pytest.raises(ValueError, match="holds 4 pages, 5"):
        c.prefix(2, 20)
    c.release(2), c.release(3)
    assert not c._prefixes


def _layer(window):
    """An attention layer whose projections are never reached."""
    layer = attention.AttentionLayer.__new__(attention.AttentionLayer)
    layer.window, layer.q_heads, layer.kv_heads, layer.head_dim = window, 2, 2, 16
    return layer


def test_windows_are_refused_where_slots_are_not_in_order(monkeypatch):
    """Before a step has written anything, in any layer."""
    class Reached(Exception):
        pass

    def reached(*a, **k):
        raise Reached

    for name in ("rms_norm", "rope_append", "linear", "paged_attention", "prefix_attention",
                 "attention_mass"):
        monkeypatch.setattr(K, name, reached)
    monkeypatch.setattr(K, "cache_evict", lambda *a, **k: a[3])
    monkeypatch.setattr(attention.AttentionLayer, "_buffers", reached)
    caches = [PagedKVCache(8, 4, 2, 16, max_seqs=3, device="cpu", track=True) for _ in range(2)]
    x, t = torch.zeros(2, 64), torch.zeros(2, dtype=torch.int32)
    pages, q = torch.zeros(1, dtype=torch.int32), torch.zeros(2, 2, 16)
    plain, windowed = _layer(0), _layer(5)
    stack = StackedMoE([None, None], [None, None], attention=[plain, windowed],
                       attention_norms=[None, None])
    step = dict(caches=caches, positions=t, seq_lens=t)

    def calls(**more):
        return (lambda: windowed.forward(x, caches[1], t, t, **more),
                lambda: stack.forward(x, **step, slots=more.get("slots"),
                                      prefixes=[more["prefix"]] * 2 if "prefix" in more else None))
    for call in calls(slots=t) + calls(prefix=pages):
        with pytest.raises(ValueError, match="window"):
            call()
    # these go through: no window; windows where nothing was cut; None for the layer with a window
    for call in calls() + (lambda: plain.forward(x, caches[0], t, t, slots=t),
                           lambda: stack.forward(x, **step, prefixes=[pages, None]),
                           lambda: caches[1].attend(q, t, window=3),
                           lambda: caches[1].weigh(q, t, q[..., 0], window=3)):
        with pytest.raises(Reached):
            call()
    assert attention.evict(caches, t, 4) is t
    for call in calls() + (lambda: caches[1].attend(q, t, window=3),
                           lambda: caches[1].weigh(q, t, q[..., 0], window=3)):
        with pytest.raises(ValueError, match="eviction: sequence 0 has been cut"):
            call()
    with pytest.raises(Reached):
        caches[1].attend(q, t)                      # no window
    caches[1].release(0)
    with pytest.raises(ValueError, match="sequence 1 has"):
        caches[1].attend(q, t, window=3)
    with pytest.raises(Reached):                    # its row is not among these
        caches[1].attend(q[:1], t[:1], window=3)
    caches[1].trim(1, 1)
    with pytest.raises(ValueError, match="sequence 1 has"):
        caches[1].attend(q, t, window=3)
    caches[1].release(1)
    for call in calls():
        with pytest.raises(Reached):
            call()


def test_lists_of_prefixes_keep_their_memory():
    """A captured step may hold a list's address behind the last release: lists are used again,
    never given back, and there are no more of a length than were in use at a time."""
    c = PagedKVCache(12, 4, 2, 16, max_seqs=4, max_pages_per_seq=6, device="cpu")
    seen = set()
    for i in range(6):
        c.reserve(i % 3, 12 + 4 * (i % 2))
        c.share(3, i % 3, 8)
        pages = c.prefix(3, 8)
        assert pages.tolist() == c._held[3][:2] and c.prefix(i % 3, 8) is pages
        assert c.prefix(i % 3, 12).tolist() == c._held[i % 3][:3]
        seen.add(pages.data_ptr())
        c.release(i % 3)
        assert pages.tolist() == c._held[3]         # still in use
        c.release(3)
    assert len(seen) == 1 and not c._prefixes
    assert {n: len(x) for n, x in c._spare.items()} == {2: 1, 3: 1}
    c.reserve(0, 8), c.reserve(1, 8)
    a, b = c.prefix(0, 8), c.prefix(1, 8)
    assert a.data_ptr() != b.data_ptr() and a.tolist() == c._held[0] and b.tolist() == c._held[1]

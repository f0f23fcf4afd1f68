"""Host side of the attention half: refusals of the C entries before any
device work, the ctypes mirror of the cache, the page bookkeeping."""
import ctypes
import os
import re

import pytest
import torch

from linuxnightmaresuite_b200 import _lib, kernels as K
from linuxnightmaresuite_b200.attention import PagedKVCache

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include",
                      "moe_b200.h")
P = ctypes.c_void_p(256)      # an aligned address that no refused call follows


@pytest.fixture(scope="module")
def lib():
    from linuxnightmaresuite_b200 import build
    build.build()
    return _lib.load()


def cache(**kw):
    a = dict(k=256, v=256, block_table=256, page_stride=16 * 2 * 64, token_stride=2 * 64,
             head_stride=64, table_stride=8, dtype=0, pages=10, page_size=16, kv_heads=2,
             head_dim=64, seqs=4, table_width=8, k_scale=1.0, v_scale=1.0)
    a.update(kw)
    return _lib.MoEPagedCache(**a)


def test_cache_mirror_matches_header():
    src = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    body = re.search(r"typedef struct moe_paged_cache \{(.*?)\} moe_paged_cache;", src, re.S)
    fields = []
    for line in body.group(1).split(";"):
        names = re.sub(r"^\s*(const\s+)?(void|int32_t|int64_t|int|float)\b", "", line).strip()
        fields += [n.strip(" *") for n in names.split(",") if n.strip()]
    assert fields == [f[0] for f in _lib.MoEPagedCache._fields_]
    enum = re.search(r"enum \{ (MOE_CACHE_F16[^}]*)\}", src, re.S).group(1)
    for name, value in re.findall(r"(MOE_CACHE_\w+)\s*=\s*(\d+)", enum):
        assert getattr(_lib, name) == int(value)
    bits = re.search(r"enum \{ (MOE_STATUS_BAD_EXPERT_ID[^}]*)\}", src, re.S).group(1)
    for name, value in re.findall(r"(MOE_STATUS_\w+)\s*=\s*(\d+)", bits):
        assert getattr(_lib, name) == int(value)
    kinds = re.search(r"enum \{\s*MOE_K_ROUTER(.*?)MOE_K_COUNT", src, re.S).group(0)
    assert len(re.findall(r"MOE_K_\w+", kinds)) - 1 == len(_lib.KERNEL_NAMES)


BAD_CACHES = [
    (dict(dtype=3), "UNSUPPORTED", "cache type"),
    (dict(k=0), "INVALID", "null"),
    (dict(block_table=0), "INVALID", "null"),
    (dict(pages=0), "INVALID", "shape"),
    (dict(page_size=0), "INVALID", "shape"),
    (dict(kv_heads=0), "INVALID", "shape"),
    (dict(seqs=-1), "INVALID", "shape"),
    (dict(table_width=0), "INVALID", "shape"),
    (dict(table_width=1 << 28), "UNSUPPORTED", "longer than"),
    (dict(head_dim=0), "UNSUPPORTED", "head_dim"),
    (dict(head_dim=60), "UNSUPPORTED", "head_dim"),
    (dict(head_dim=264), "UNSUPPORTED", "head_dim"),
    (dict(dtype=2, head_dim=72), "UNSUPPORTED", "head_dim"),
    (dict(k=264), "INVALID", "16 bytes"),
    (dict(token_stride=132), "INVALID", "16 bytes"),
    (dict(page_stride=-2048), "INVALID", "negative"),
    (dict(k_scale=0.5), "INVALID", "scales"),
    (dict(dtype=2, k_scale=0.0), "INVALID", "scales"),
    (dict(dtype=2, v_scale=float("nan")), "INVALID", "scales"),
]


def attention(lib, c, q=P, lens=P, hq=4, max_len=0, window=0, scale=0.1, cap=0.0, out=P, ws=P,
              nbytes=1 << 26):
    return lib.moe_paged_attention(ctypes.byref(c), q, 256, 64, lens, hq, max_len, window, scale,
                                   cap, out, None, ws, nbytes, None)


def append(lib, c, q=P, k=P, v=P, T=2, hq=4, pos=P, seq=None, freq=P, rot=64, q_out=P):
    return lib.moe_rope_append(ctypes.byref(c), q, 256, 64, k, 128, 64, v, 128, 64, T, hq, pos,
                               seq, freq, rot, 0, q_out, 256, 64, None, None)


@pytest.mark.parametrize("change,status,words", BAD_CACHES)
def test_bad_caches_are_refused(lib, change, status, words):
    c = cache(**change)
    for call in (attention, append):
        assert call(lib, c) == getattr(_lib, "MOE_ERR_" + status)
        assert words in _lib.last_error()


def test_bad_attention_arguments_are_refused(lib):
    c = cache()
    for kw, status in ((dict(hq=0), "INVALID"), (dict(hq=5), "INVALID"),
                       (dict(max_len=-1), "INVALID"), (dict(window=-1), "INVALID"),
                       (dict(cap=-1.0), "INVALID"), (dict(cap=float("inf")), "INVALID"),
                       (dict(scale=float("nan")), "INVALID"), (dict(q=None), "INVALID"),
                       (dict(lens=None), "INVALID"), (dict(out=None), "INVALID"),
                       (dict(ws=None), "INVALID"), (dict(nbytes=16), "WORKSPACE")):
        assert attention(lib, c, **kw) == getattr(_lib, "MOE_ERR_" + status), kw
    assert attention(lib, cache(seqs=0), q=None) == _lib.MOE_OK       # nothing to do
    assert lib.moe_paged_attention(None, P, 1, 1, P, 4, 0, 0, 0.1, 0.0, P, None, P, 1 << 26,
                                   None) == _lib.MOE_ERR_INVALID
    n = ctypes.c_size_t()
    assert lib.moe_paged_attention_workspace_bytes(4, 4, 2, 64, ctypes.byref(n)) == _lib.MOE_OK
    assert n.value >= 256
    for bad in ((-1, 4, 2, 64), (4, 5, 2, 64), (4, 4, 0, 64), (4, 4, 2, 257)):
        assert lib.moe_paged_attention_workspace_bytes(*bad, ctypes.byref(n)) == \
            _lib.MOE_ERR_INVALID


def test_bad_append_arguments_are_refused(lib):
    c = cache()
    for kw in (dict(T=-1), dict(hq=-1), dict(rot=3), dict(rot=66), dict(rot=-2), dict(k=None),
               dict(v=None), dict(pos=None), dict(freq=None), dict(q=None), dict(q_out=None),
               dict(T=5)):
        assert append(lib, c, **kw) == _lib.MOE_ERR_INVALID, kw
    assert append(lib, c, T=0, k=None) == _lib.MOE_OK
    assert lib.moe_rope_append(None, P, 1, 1, P, 1, 1, P, 1, 1, 1, 1, P, None, P, 64, 0, P, 1, 1,
                               None, None) == _lib.MOE_ERR_INVALID


def test_bad_linear_arguments_are_refused(lib):
    def lin(w=P, qt=2, rows=64, cols=64, x=P, T=1, y=P):
        return lib.moe_linear(w, qt, rows, cols, x, 64, T, None, 0, y, 64, None)
    for kw, status in ((dict(qt=12), "UNSUPPORTED"), (dict(cols=48), "UNSUPPORTED"),
                       (dict(rows=0), "INVALID"), (dict(cols=0), "INVALID"),
                       (dict(T=-1), "INVALID"), (dict(w=None), "INVALID"),
                       (dict(x=None), "INVALID"), (dict(y=None), "INVALID"),
                       (dict(w=ctypes.c_void_p(264)), "INVALID")):
        assert lin(**kw) == getattr(_lib, "MOE_ERR_" + status), kw
    assert lin(T=0, x=None) == _lib.MOE_OK


def test_wrappers_refuse_host_tensors():
    k = torch.zeros((2, 4, 1, 64), dtype=torch.float16)
    t = torch.zeros((1, 2), dtype=torch.int32)
    with pytest.raises(TypeError, match="CUDA"):
        K.paged_attention(torch.zeros(1, 2, 64), k, k, t, t[0, :1])
    with pytest.raises(TypeError, match="CUDA"):
        K.rope_append(None, k[:, 0], k[:, 0], k, k, t, t[0, :1])
    with pytest.raises(TypeError, match="CUDA"):
        K.LinearWeights(torch.zeros(18, dtype=torch.uint8), 2, 1, 32)
    with pytest.raises(ValueError):
        K.rope_inv_freq(7)
    f = K.rope_inv_freq(8, 10000.0, torch.tensor([1.0, 1.0, 2.0, 4.0]), device="cpu")
    assert f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.005, 0.00025], dtype=torch.float64))


def test_pages_are_handed_out_and_come_back():
    c = PagedKVCache(6, 4, 2, 16, max_seqs=3, max_pages_per_seq=4, device="cpu")
    address = c.block_table.data_ptr()
    c.reserve(0, 1)
    c.reserve(0, 4)
    assert c.free_pages == 5
    c.reserve(0, 5)
    c.reserve(2, 16)
    assert c.free_pages == 0
    held = c.block_table[0, :2].tolist() + c.block_table[2].tolist()
    assert sorted(held) == list(range(6))
    assert (c.block_table[1] == -1).all() and (c.block_table[0, 2:] == -1).all()
    with pytest.raises(RuntimeError, match="full"):
        c.reserve(1, 1)
    with pytest.raises(ValueError, match="at most 4"):
        c.reserve(2, 17)
    with pytest.raises(IndexError):
        c.reserve(3, 1)
    c.release(2)
    assert c.free_pages == 4 and (c.block_table[2] == -1).all()
    c.reserve(1, 16)
    assert c.free_pages == 0
    assert sorted(c.block_table[0, :2].tolist() + c.block_table[1].tolist()) == list(range(6))
    c.reserve(1, 0)
    c.reserve(1, -3)
    assert c.block_table.data_ptr() == address
    with pytest.raises(TypeError):
        PagedKVCache(1, 1, 1, 16, 1, dtype=torch.float32, device="cpu")
    with pytest.raises(ValueError):
        PagedKVCache(0, 1, 1, 16, 1, device="cpu")
    e = PagedKVCache(2, 4, 1, 16, 1, dtype=torch.float8_e4m3fn, device="cpu")
    assert e.k.view(torch.uint8).sum() == 0


@pytest.mark.parametrize("name, mirror", [
    ("moe_rope_append_args", _lib.MoERopeAppendArgs),
    ("moe_paged_attention_args", _lib.MoEPagedAttentionArgs),
    ("moe_linear_args", _lib.MoELinearArgs)])
def test_argument_record_matches_header(name, mirror):
    src = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), src, re.S).group(1)
    size = {"int": 4, "float": 4}
    fields = []
    for line in body.split(";"):
        m = re.match(r"\s*(?:const\s+)?(\w+)\s*(\*?)(.*)", line, re.S)
        if m is None:
            continue
        for n in m.group(3).split(","):
            star = bool(m.group(2)) or "*" in n
            fields.append((n.strip(" *\n"), None if m.group(1) == "moe_paged_cache" else
                           8 if star else size.get(m.group(1), 8)))
    import ctypes
    assert [f for f, _ in fields] == [f[0] for f in mirror._fields_]
    assert all(b is None or b == ctypes.sizeof(f[1]) for (_, b), f in zip(fields, mirror._fields_))


def test_records_reach_the_same_checks(lib):
    """The record forms refuse and accept what the calls do."""
    import ctypes
    for n in ("moe_rope_append_record", "moe_paged_attention_record", "moe_linear_record"):
        assert getattr(lib, n)(None) == _lib.MOE_ERR_INVALID
        assert "null arguments" in _lib.last_error()
    a = _lib.MoEPagedAttentionArgs(cache=cache(), q=256, q_seq_stride=256, q_head_stride=64,
                                   seq_lens=256, out=256, lse=0, workspace=256,
                                   workspace_bytes=1, stream=0, q_heads=4, max_len=0, window=0,
                                   scale=0.1, softcap=0.0)
    assert lib.moe_paged_attention_record(ctypes.byref(a)) == _lib.MOE_ERR_WORKSPACE
    a.q_heads = 3
    assert lib.moe_paged_attention_record(ctypes.byref(a)) == _lib.MOE_ERR_INVALID
    a.cache.seqs, a.q_heads = 0, 4
    assert lib.moe_paged_attention_record(ctypes.byref(a)) == _lib.MOE_OK
    r = _lib.MoERopeAppendArgs(cache=cache(), T=0, q_heads=4, rot=64)
    assert lib.moe_rope_append_record(ctypes.byref(r)) == _lib.MOE_OK
    r.rot = 63
    assert lib.moe_rope_append_record(ctypes.byref(r)) == _lib.MOE_ERR_INVALID
    w = _lib.MoELinearArgs(qtype=_lib.MOE_Q4_0, rows=16, cols=64, T=0)
    assert lib.moe_linear_record(ctypes.byref(w)) == _lib.MOE_OK
    w.cols = 65
    assert lib.moe_linear_record(ctypes.byref(w)) == _lib.MOE_ERR_UNSUPPORTED


def test_slots_that_share_memory_are_refused(lib):
    """A token stride of 0 with several slots per page: the tensor map of the
    attention cannot hold it, an append would write its slots over one another.
    Rows closer than head_dim are nothing to append to either."""
    for kw in (dict(token_stride=0), dict(token_stride=0, page_stride=128, pages=2)):
        for call in (attention, append):
            assert call(lib, cache(**kw)) == _lib.MOE_ERR_INVALID, kw
            assert "share memory" in _lib.last_error()
    for kw in (dict(page_stride=0), dict(head_stride=0), dict(head_stride=56), dict(token_stride=8),
               dict(page_stride=32)):
        assert append(lib, cache(**kw)) == _lib.MOE_ERR_INVALID, kw
        assert "share memory" in _lib.last_error()
    # one slot, one head, one page: no stride that counts; T = 0 stops behind the checks
    assert append(lib, cache(page_size=1, token_stride=0), T=0) == _lib.MOE_OK
    assert append(lib, cache(kv_heads=1, head_stride=0), T=0) == _lib.MOE_OK
    assert append(lib, cache(pages=1, page_stride=0), T=0) == _lib.MOE_OK
    # the attention only reads: one head for all, one page for all
    for kw in (dict(page_stride=0), dict(head_stride=0)):
        assert attention(lib, cache(**kw), ws=None) == _lib.MOE_ERR_INVALID
        assert "null pointer" in _lib.last_error()


def test_workspace_off_its_alignment_is_refused(lib):
    """Parts of units are fetched from the workspace by bulk copies, whose source
    must lie on 16 bytes."""
    for at in (257, 260, 264):
        assert attention(lib, cache(), ws=ctypes.c_void_p(at)) == _lib.MOE_ERR_INVALID
        assert "16-byte" in _lib.last_error()


@pytest.mark.parametrize("axis", [dict(pages=1, page_stride=3), dict(page_size=1, token_stride=-5),
                                  dict(kv_heads=1, head_stride=7),
                                  dict(pages=1, page_stride=1, page_size=1, token_stride=-1,
                                       kv_heads=1, head_stride=0)])
def test_strides_of_single_axes_are_ignored(lib, axis):
    c = cache(**axis)
    assert append(lib, c, T=0) == _lib.MOE_OK
    assert attention(lib, c, ws=None) == _lib.MOE_ERR_INVALID    # behind the cache's checks
    assert "null pointer" in _lib.last_error()


def test_linear_rows_that_overlap_are_refused(lib):
    """y is written while x is still read.  The calls that pass the check are too
    wide for any kernel, so nothing is launched."""
    cols, rows, base = 1 << 21, 1 << 20, 1 << 40

    def lin(x=0, xs=cols, y=1 << 30, ys=rows, T=1, res=None, rs=0):
        at = [None if e is None else ctypes.c_void_p(base + 4 * e) for e in (x, y, res)]
        return lib.moe_linear(P, 2, rows, cols, at[0], xs, T, at[2], rs, at[1], ys, None)
    both = cols + rows                              # x and y side by side in one buffer
    for kw in (dict(y=0), dict(y=cols - 1), dict(y=1 - rows), dict(y=0, T=3, ys=both, xs=both),
               dict(y=3 * cols, T=4), dict(y=cols - 1, T=3, ys=both, xs=both),
               dict(T=2, ys=rows - 1), dict(T=2, ys=0),                       # rows of y
               dict(res=(1 << 30) + 1), dict(res=(1 << 30) - rows + 1),       # residual
               dict(res=1 << 30, rs=rows + 8, T=2), dict(res=(1 << 30) + rows, rs=rows, T=2)):
        assert lin(**kw) == _lib.MOE_ERR_INVALID, kw
        assert "overlap" in _lib.last_error()
    for kw in (dict(), dict(y=cols), dict(y=-rows), dict(y=cols, T=3, xs=both, ys=both),
               dict(y=-rows, T=3, xs=both, ys=both), dict(xs=0, T=5), dict(T=1, ys=0),
               dict(y=cols, T=2, xs=2 * both, ys=2 * both),
               dict(res=1 << 30, rs=rows, T=2), dict(res=1 << 30, rs=7), dict(res=0, rs=rows, T=2),
               dict(res=(1 << 30) + rows), dict(res=(1 << 30) + rows, rs=2 * rows, T=2, ys=2 * rows)):
        assert lin(**kw) not in (_lib.MOE_ERR_INVALID, _lib.MOE_OK), (kw, _lib.last_error())
        assert "overlap" not in _lib.last_error()


def test_rotated_q_that_overlaps_is_refused(lib):
    def rope(q=1024, k=4096, v=8192, out=1024, qs=(256, 64), os=(256, 64), T=2, hq=4):
        at = [ctypes.c_void_p(a) for a in (q, k, v, out)]
        return lib.moe_rope_append(ctypes.byref(cache()), at[0], *qs, at[1], 128, 64, at[2], 128,
                                   64, T, hq, P, None, P, 64, 0, at[3], *os, None, None)
    for kw in (dict(out=4096), dict(out=8192), dict(out=2048, os=(0, 64)),
               dict(out=2048, os=(256, 0)), dict(out=2048, os=(256, 60)), dict(os=(512, 64)),
               dict(os=(256, 128)), dict(qs=(0, 64))):
        assert rope(**kw) == _lib.MOE_ERR_INVALID, kw
        assert "q_out" in _lib.last_error()


def test_no_sequences_need_no_table(lib):
    """An empty tensor has no address."""
    empty = cache(seqs=0, block_table=0)
    assert attention(lib, empty, q=None) == _lib.MOE_OK
    assert append(lib, empty, T=0) == _lib.MOE_OK
    assert attention(lib, cache(block_table=0)) == _lib.MOE_ERR_INVALID


def test_status_is_read_on_its_own_device(monkeypatch):
    """The copy of a status word goes behind the kernels of the device that it is on."""
    current, seen = [0], []

    class On:
        def __init__(self, device):
            self.device = torch.device(device).index

        def __enter__(self):
            current.append(self.device)

        def __exit__(self, *_):
            current.pop()

    class Lib:
        @staticmethod
        def moe_read_status(ws, out, stream):
            seen.append(current[-1])
            return _lib.MOE_OK
    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(_lib, "load", lambda: Lib)
    monkeypatch.setattr(K, "_stream", lambda: None)
    ws = type("T", (), dict(device=torch.device("cuda", 3), data_ptr=lambda self: 256))()
    assert K.read_status(ws) == 0 and seen == [3]


def test_attention_output_over_part_of_q_is_refused(lib):
    c = cache()                                     # 4 sequences of 4 heads of 64: 4096 bytes

    def att(q, out, ss=256, hs=64):
        return lib.moe_paged_attention(ctypes.byref(c), ctypes.c_void_p(q), ss, hs, P, 4, 0, 0, 0.1,
                                       0.0, ctypes.c_void_p(out), None, P, 16, None)
    q = 1 << 20
    for out, strides in ((q + 4, {}), (q - 4, {}), (q + 4092, {}), (q - 4092, {}), (q + 1024, {}),
                         (q, dict(ss=512)), (q, dict(hs=128)), (q + 1024, dict(ss=512)),
                         (q, dict(ss=0))):
        assert att(q, out, **strides) == _lib.MOE_ERR_INVALID, (out - q, strides)
        assert "overlap" in _lib.last_error()
    for out, strides in ((q, {}), (q + 4096, {}), (q - 4096, {}), (q - 4096, dict(ss=512)),
                         (q + 4 * (3 * 512 + 256), dict(ss=512))):
        assert att(q, out, **strides) == _lib.MOE_ERR_WORKSPACE, (out - q, strides)

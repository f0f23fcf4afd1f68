"""Torch-tensor wrappers over the C ABI.

Every function takes CUDA tensors, allocates outputs and workspaces with torch
and enqueues the library's kernels on the current CUDA stream.  Inputs that
are not contiguous CUDA tensors of the right dtype are rejected.
"""
from __future__ import annotations

import ctypes
import struct
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import call, entry

QTYPE_F32 = _lib.MOE_F32
QTYPE_Q4_0 = _lib.MOE_Q4_0
QTYPE_Q5_1 = _lib.MOE_Q5_1
QTYPE_Q8_0 = _lib.MOE_Q8_0
QTYPE_Q4_K = _lib.MOE_Q4_K
QTYPE_Q6_K = _lib.MOE_Q6_K
ACT_SWIGLU = _lib.MOE_ACT_SWIGLU
ACT_GEGLU_TANH = _lib.MOE_ACT_GEGLU_TANH
KERNELS_AUTO = _lib.MOE_KERNELS_AUTO
KERNELS_GEMV = _lib.MOE_KERNELS_GEMV
KERNELS_BLOCKSCALE = _lib.MOE_KERNELS_BLOCKSCALE
KERNELS_SPLIT_GEMM = _lib.MOE_KERNELS_SPLIT_GEMM
STATUS_BAD_PAGE = _lib.MOE_STATUS_BAD_PAGE
# GGML type -> (weights per block, bytes per block), dequant_fast.py:723-754
BLOCK_GEOMETRY = {QTYPE_F32: (1, 4), QTYPE_Q4_0: (32, 18), QTYPE_Q5_1: (32, 24),
                  QTYPE_Q8_0: (32, 34), QTYPE_Q4_K: (256, 144), QTYPE_Q6_K: (256, 210)}
BLOCK_BYTES = {QTYPE_Q4_0: 18, QTYPE_Q8_0: 34}
PACKED_QTYPES = (QTYPE_Q4_0, QTYPE_Q8_0)


def row_bytes(qtype: int, cols: int) -> int:
    e, b = BLOCK_GEOMETRY[qtype]
    if cols % e:
        raise ValueError(f"row of {cols} weights is not whole blocks of type {qtype}")
    return cols // e * b


def packed_path(qtype: int, down_qtype: int) -> bool:
    """Whether a layer's expert matrices are repacked into MMA tiles (Q4_0 /
    Q8_0 on all three) or used as stored (every other combination)."""
    return qtype in PACKED_QTYPES and down_qtype == qtype


class ExpertOpts:
    """Expert variant (``moe_expert_opts``): activation, down matrix type,
    gate/up stride of a fused stack, per-expert down scale (device f32), and
    the kernel family (``KERNELS_*``, 0 = automatic) with its chunk rows."""

    def __init__(self, act: int = ACT_SWIGLU, down_qtype: int = 0, gate_up_stride: int = 0,
                 down_scale: Optional[torch.Tensor] = None, kernels: int = 0,
                 chunk_rows: int = 0):
        if down_scale is not None:
            _need(down_scale, torch.float32, "down_scale")
        self.down_scale = down_scale
        self.c = _lib.MoEExpertOpts(act, down_qtype, gate_up_stride,
                                    0 if down_scale is None else down_scale.data_ptr(),
                                    kernels, chunk_rows)

    @property
    def ref(self):
        return ctypes.byref(self.c)


def _stream() -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _ptr(t: Optional[torch.Tensor]):
    return ctypes.c_void_p(0 if t is None else t.data_ptr())


def _need(t: torch.Tensor, dtype, name: str, pinned_ok: bool = False) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or not (t.is_cuda or (pinned_ok and t.is_pinned())):
        raise TypeError(f"{name} must be a CUDA tensor" + (" or pinned host memory"
                                                          if pinned_ok else ""))
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def _size_out(fn: str, *args) -> int:
    out = ctypes.c_size_t(0)
    call(fn, *args, ctypes.byref(out))
    return int(out.value)


def workspace(nbytes: int, device) -> torch.Tensor:
    return torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=device)


class RowBuffers:
    """f32 scratch rows of an object that is called with any number of rows.  A
    captured CUDA graph holds the addresses that its calls used, so no buffer is
    ever replaced: there is one for each power of two of rows (at most twice the
    largest in all), and a call uses the first rows of the one that fits."""

    def __init__(self):
        self._buffers = {}
        self._rows = {}

    def rows(self, T: int, width: int, device) -> torch.Tensor:
        """(T, width), the same memory at every call."""
        key = (T, width, device)
        t = self._rows.get(key)
        if t is None:
            whole = (1 << max(T - 1, 0).bit_length(), width, device)
            buf = self._buffers.get(whole)
            if buf is None:
                buf = self._buffers[whole] = torch.empty(whole[:2], dtype=torch.float32,
                                                         device=device)
            t = self._rows[key] = buf[:T]
        return t


def block_geometry(qtype: int) -> Tuple[int, int]:
    e, b = ctypes.c_int(0), ctypes.c_int(0)
    call("moe_block_geometry", qtype, ctypes.byref(e), ctypes.byref(b))
    return e.value, b.value


# --------------------------------------------------------------------------- weights

def router_input(x: torch.Tensor, scale: Optional[torch.Tensor], eps: float = 1e-6,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """gemma4's router input, x / sqrt(mean(x^2) + eps) * f32(1/sqrt(d)) * scale
    (nightmare_stream.py:4662-4667)."""
    _need(x, torch.float32, "x")
    if scale is not None:
        _need(scale, torch.float32, "scale")
    T, d = x.shape
    if out is None:
        out = torch.empty_like(x)
    call("moe_router_input", _ptr(x), _ptr(scale), ctypes.c_float(eps), T, d, _ptr(out),
         _stream())
    return out


def dequantize(raw: torch.Tensor, qtype: int, n_elements: int) -> torch.Tensor:
    _need(raw, torch.uint8, "raw")
    out = torch.empty(n_elements, dtype=torch.float32, device=raw.device)
    call("moe_dequantize", _ptr(raw), _ptr(out), qtype, n_elements, _stream())
    return out


def pack_weights(raw: torch.Tensor, qtype: int, n_mats: int, rows: int, cols: int) -> torch.Tensor:
    _need(raw, torch.uint8, "raw")
    nbytes = _size_out("moe_packed_bytes", qtype, n_mats, rows, cols)
    if raw.numel() != nbytes:
        raise ValueError(f"raw blocks hold {raw.numel()} bytes, expected {nbytes}")
    out = torch.empty(nbytes, dtype=torch.uint8, device=raw.device)
    call("moe_pack_weights", _ptr(raw), _ptr(out), qtype, n_mats, rows, cols, _stream())
    return out


def unpack_weights(packed: torch.Tensor, qtype: int, n_mats: int, rows: int, cols: int) -> torch.Tensor:
    _need(packed, torch.uint8, "packed")
    out = torch.empty_like(packed)
    call("moe_unpack_weights", _ptr(packed), _ptr(out), qtype, n_mats, rows, cols, _stream())
    return out


# --------------------------------------------------------------------------- stages

def router(x: torch.Tensor, gate_w: torch.Tensor, k: int, mode: int = 0,
           bias: Optional[torch.Tensor] = None, layout: int = _lib.MOE_ROUTER_D_E):
    """(ids int32 (T,k), weights f32 (T,k)) for x (T, d)."""
    _need(x, torch.float32, "x")
    _need(gate_w, torch.float32, "gate_w")
    if bias is not None:
        _need(bias, torch.float32, "bias")
    T, d = x.shape
    E = gate_w.shape[1] if layout == _lib.MOE_ROUTER_D_E else gate_w.shape[0]
    ids = torch.empty((T, k), dtype=torch.int32, device=x.device)
    w = torch.empty((T, k), dtype=torch.float32, device=x.device)
    ws = workspace(_size_out("moe_router_workspace_bytes", T, d, E), x.device)
    call("moe_router", _ptr(x), _ptr(gate_w), _ptr(bias), T, d, E, k, layout, mode,
         _ptr(ids), _ptr(w), _ptr(ws), ws.numel(), _stream())
    return ids, w


def dispatch(ids: torch.Tensor, n_experts: int, ws: Optional[torch.Tensor] = None):
    """(expert_offsets (E+1), perm_rows (T*k), inv_perm (T*k)), all int32."""
    _need(ids, torch.int32, "ids")
    T, k = ids.shape
    dev = ids.device
    off = torch.empty(n_experts + 1, dtype=torch.int32, device=dev)
    perm = torch.empty(T * k, dtype=torch.int32, device=dev)
    inv = torch.empty(T * k, dtype=torch.int32, device=dev)
    if ws is None:
        ws = workspace(_size_out("moe_dispatch_workspace_bytes", T, k, n_experts), dev)
        ws[:256].zero_()
    call("moe_dispatch", _ptr(ids), T, k, n_experts, _ptr(off), _ptr(perm), _ptr(inv),
         _ptr(ws), ws.numel(), _stream())
    return off, perm, inv


def read_status(ws: torch.Tensor) -> int:
    """Reads and clears a workspace's status bits, behind what its device's
    current stream holds (synchronises)."""
    st = ctypes.c_int(0)
    with torch.cuda.device(ws.device):
        rc = _lib.load().moe_read_status(_ptr(ws), ctypes.byref(st), _stream())
    if rc not in (_lib.MOE_OK, _lib.MOE_ERR_DEVICE):
        _lib.check(rc)
    return st.value


def experts(w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, qtype: int,
            offsets: torch.Tensor, x: torch.Tensor, d: int, F: int,
            x_rows: Optional[torch.Tensor] = None, x_rows_div: int = 1,
            y: Optional[torch.Tensor] = None, y_rows: Optional[torch.Tensor] = None,
            rows: Optional[int] = None, ws: Optional[torch.Tensor] = None,
            opts: Optional[ExpertOpts] = None) -> torch.Tensor:
    """Grouped experts on packed weights (Q4_0 / Q8_0) or raw matrices (other
    types, or a down matrix of another type); returns y (rows, d) f32."""
    for t, n in ((w_gate, "w_gate"), (w_up, "w_up"), (w_down, "w_down")):
        if not isinstance(t, torch.Tensor) or not t.is_cuda or not t.is_contiguous():
            raise TypeError(f"{n} must be a contiguous CUDA tensor")
    _need(offsets, torch.int32, "offsets")
    _need(x, torch.float32, "x")
    E = offsets.numel() - 1
    if rows is None:
        rows = int(offsets[-1].item())
    if y is None:
        y = torch.empty((rows, d), dtype=torch.float32, device=x.device)
    if ws is None:
        ws = workspace(_size_out("moe_experts_workspace_bytes", rows, E, d, F), x.device)
        ws[:256].zero_()
    call("moe_experts_ex", _ptr(w_gate), _ptr(w_up), _ptr(w_down), qtype,
         None if opts is None else opts.ref, _ptr(offsets), E, rows, _ptr(x), _ptr(x_rows),
         x_rows_div, d, F, _ptr(y), _ptr(y_rows), _ptr(ws), ws.numel(), _stream())
    return y


def combine(y: torch.Tensor, inv_perm: torch.Tensor, weights: torch.Tensor,
            shared: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    T, k = weights.shape
    d = y.shape[1]
    if out is None:
        out = torch.empty((T, d), dtype=torch.float32, device=y.device)
    call("moe_combine", _ptr(y), _ptr(inv_perm), _ptr(weights), _ptr(shared), _ptr(residual),
         T, k, d, _ptr(out), _stream())
    return out


def gather_rows(x: torch.Tensor, rows: torch.Tensor, div: int = 1,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    _need(x, torch.float32, "x")
    _need(rows, torch.int32, "rows")
    n, d = rows.numel(), x.shape[1]
    if out is None:
        out = torch.empty((n, d), dtype=torch.float32, device=x.device)
    call("moe_gather_rows", _ptr(x), _ptr(rows), div, n, d, _ptr(out), _stream())
    return out


def ep_local_order(recv_counts: torch.Tensor, max_rows: int, ws: torch.Tensor):
    """(local_offsets (E_local+1), row_map (max_rows)) on the device."""
    _need(recv_counts, torch.int32, "recv_counts")
    W, El = recv_counts.shape
    loff = torch.empty(El + 1, dtype=torch.int32, device=recv_counts.device)
    row_map = torch.empty(max(max_rows, 1), dtype=torch.int32, device=recv_counts.device)
    call("moe_ep_local_order", _ptr(recv_counts), W, El, max_rows, _ptr(loff), _ptr(row_map),
         _ptr(ws), _stream())
    return loff, row_map


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
             out: Optional[torch.Tensor] = None, gemma_style: bool = False) -> torch.Tensor:
    _need(x, torch.float32, "x")
    _need(weight, torch.float32, "weight")
    T, d = x.shape
    if out is None:
        out = torch.empty_like(x)
    call("moe_rms_norm_ex", _ptr(x), _ptr(weight), ctypes.c_float(eps), 1 if gemma_style else 0,
         T, d, _ptr(out), _stream())
    return out


# --------------------------------------------------------------------------- attention half

CACHE_TYPES = {torch.float16: _lib.MOE_CACHE_F16, torch.bfloat16: _lib.MOE_CACHE_BF16,
               torch.float8_e4m3fn: _lib.MOE_CACHE_E4M3}


# The arguments as the entry points read them (moe_*_args), packed in one step:
# a ctypes call converts each argument at the price of packing five.
_CACHE = "3P4q7i2f"
_APPEND_ARGS = struct.Struct("@" + _CACHE + "3P6q4P2q2P4i0q")
_ATTENTION_ARGS = struct.Struct("@" + _CACHE + "P2q4PNP3i2f0q")
_LINEAR_ARGS = struct.Struct("@2PqPqPqP4i")
assert _APPEND_ARGS.size == ctypes.sizeof(_lib.MoERopeAppendArgs)
assert _ATTENTION_ARGS.size == ctypes.sizeof(_lib.MoEPagedAttentionArgs)
assert _LINEAR_ARGS.size == ctypes.sizeof(_lib.MoELinearArgs)


def _enqueue(name: str, index: int, args: bytes) -> None:
    """The entry point, with device ``index`` current."""
    fn = entry(name)
    if index == _current_device():
        rc = fn(args)
    else:
        with torch.cuda.device(index):
            rc = fn(args)
    if rc:
        _lib.check(rc)


# These wrappers are called once per layer and token, on kernels of a few
# microseconds, so each check of an argument is one expression; what it refuses
# is told apart here.
def _refuse(t, name: str, dtype, index: int, shape=None) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, expected cuda:{index}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} is {tuple(t.shape)}, expected {tuple(shape)}")
    raise ValueError(f"{name} must be contiguous")


_F32, _I32 = torch.float32, torch.int32
_current_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream


def _rows_f32(t: torch.Tensor, name: str, index: int, shape) -> Tuple[int, ...]:
    """Strides of a CUDA f32 tensor of the shape whose last axis is contiguous;
    the other axes may stride."""
    if t.dtype is not _F32 or t.get_device() != index or t.shape != shape:
        _refuse(t, name, _F32, index, shape)
    strides = t.stride()
    if strides[-1] != 1 and shape[-1] > 1:
        raise ValueError(f"the last axis of {name} must be contiguous")
    return strides


def _vector(t: torch.Tensor, dtype, name: str, index: int, n: int) -> int:
    """Address of a contiguous CUDA vector of n elements."""
    if t.dtype is not dtype or t.get_device() != index or t.shape != (n,) or \
            not t.is_contiguous():
        _refuse(t, name, dtype, index, (n,))
    return t.data_ptr()


def _paged_cache(k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                 k_scale: float, v_scale: float):
    """(fields of a moe_paged_cache, device index, sequences, kv_heads, head_dim)."""
    index, dtype = k_cache.get_device(), k_cache.dtype
    if index < 0:
        raise TypeError("k_cache must be a CUDA tensor")
    kind = CACHE_TYPES.get(dtype)
    if kind is None:
        raise TypeError(f"caches of {dtype}: one of "
                        f"{', '.join(str(t) for t in CACHE_TYPES)} is needed")
    shape, strides = k_cache.shape, k_cache.stride()
    if v_cache.dtype is not dtype or v_cache.get_device() != index:
        _refuse(v_cache, "v_cache", dtype, index)
    if len(shape) != 4 or v_cache.shape != shape or (v_cache.stride() != strides and any(
            a != b and n > 1 for a, b, n in zip(strides, v_cache.stride(), shape))):
        raise ValueError("k_cache and v_cache must be (pages, page_size, kv_heads, head_dim) of "
                         "the same shape and strides")
    if strides[3] != 1 and shape[3] > 1:
        raise ValueError("the last axis of the caches must be contiguous")
    if block_table.dtype is not _I32 or block_table.get_device() != index:
        _refuse(block_table, "block_table", _I32, index)
    table, trow = block_table.shape, block_table.stride()
    if len(table) != 2 or (trow[1] != 1 and table[1] > 1):
        raise ValueError("block_table must be (sequences, pages of a sequence) with contiguous "
                         "rows")
    return ((k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), strides[0],
             strides[1], strides[2], trow[0], kind, *shape, *table, k_scale, v_scale),
            index, table[0], shape[2], shape[3])


def rope_append(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor,
                k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                positions: torch.Tensor, inv_freq: Optional[torch.Tensor] = None,
                seq_ids: Optional[torch.Tensor] = None, interleaved: bool = False,
                k_scale: float = 1.0, v_scale: float = 1.0, q_out: Optional[torch.Tensor] = None,
                status: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Rotates q (T, q_heads, head_dim) and k (T, kv_heads, head_dim) by their
    positions, writes k and v into the paged caches (pages, page_size,
    kv_heads, head_dim; any page layout as a view) and returns the rotated q
    (``q_out``, which may be q itself but may not share memory with k or v).

    ``inv_freq`` (rot / 2,) f64 holds the angle of each pair per position
    (``rope_inv_freq``); None rotates nothing.  Pairs are (i, i + rot / 2), or
    adjacent with ``interleaved``.  ``seq_ids`` maps tokens to rows of
    ``block_table`` (None: token t is sequence t); a negative position skips
    its token, q row included (without ``q_out`` that row is not set); no two
    tokens may share sequence and position.
    ``status`` (int32) receives STATUS_BAD_PAGE for a page or sequence that
    does not exist; such a token's k and v are not stored."""
    c, dev, _, hk, d = _paged_cache(k_cache, v_cache, block_table, k_scale, v_scale)
    T = k.shape[0]
    ks = _rows_f32(k, "k", dev, (T, hk, d))
    vs = _rows_f32(v, "v", dev, (T, hk, d))
    rot = freq = 0
    if inv_freq is not None:
        rot = 2 * inv_freq.numel()
        freq = _vector(inv_freq, torch.float64, "inv_freq", dev, inv_freq.numel())
    hq, qs, os_, q_ptr, o_ptr = 0, (0, 0), (0, 0), 0, 0
    if q is not None:
        shape = q.shape
        if len(shape) != 3:
            raise ValueError("q must be (tokens, q_heads, head_dim)")
        hq = shape[1]
        qs = _rows_f32(q, "q", dev, (T, hq, d))
        if q_out is None:
            q_out = torch.empty_like(q)          # dense, whatever q's strides
            os_ = q_out.stride()
        else:
            os_ = _rows_f32(q_out, "q_out", dev, (T, hq, d))
        q_ptr, o_ptr = q.data_ptr(), q_out.data_ptr()
    _enqueue("moe_rope_append_record", dev, _APPEND_ARGS.pack(
        *c, q_ptr, k.data_ptr(), v.data_ptr(), qs[0], qs[1], ks[0], ks[1], vs[0], vs[1],
        _vector(positions, _I32, "positions", dev, T),
        0 if seq_ids is None else _vector(seq_ids, _I32, "seq_ids", dev, T), freq, o_ptr, os_[0],
        os_[1], 0 if status is None else _vector(status, _I32, "status", dev, 1),
        _raw_stream(dev), T, hq, rot, 1 if interleaved else 0))
    return q_out


def rope_inv_freq(rot: int, base: float = 10000.0, factors: Optional[torch.Tensor] = None,
                  device=None) -> torch.Tensor:
    """(rot / 2,) f64 angles per position, base ** (-2 i / rot), divided by
    ``factors`` (a GGUF ``rope_freqs`` tensor) if given."""
    if rot <= 0 or rot % 2:
        raise ValueError(f"rot {rot} must be even and positive")
    f = float(base) ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot)
    if factors is not None:
        if factors.numel() != rot // 2:
            raise ValueError(f"{factors.numel()} factors for {rot // 2} pairs")
        f = f / factors.detach().to("cpu", torch.float64).reshape(-1)
    return f.to(device if device is not None else torch.device("cuda"))


def paged_attention_workspace(seqs: int, q_heads: int, kv_heads: int, head_dim: int,
                              device) -> torch.Tensor:
    """A workspace for ``paged_attention`` calls of these heads, with any number
    of sequences, that follow one another (calls that may overlap need one each)."""
    n = _size_out("moe_paged_attention_workspace_bytes", seqs, q_heads, kv_heads, head_dim)
    return torch.zeros(n, dtype=torch.uint8, device=device)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    block_table: torch.Tensor, seq_lens: torch.Tensor,
                    scale: Optional[float] = None, window: int = 0, softcap: float = 0.0,
                    k_scale: float = 1.0, v_scale: float = 1.0, max_len: int = 0,
                    out: Optional[torch.Tensor] = None, return_lse: bool = False,
                    ws: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None):
    """Attention of one new token per sequence, q (seqs, q_heads, head_dim),
    over the first ``seq_lens[s]`` tokens of its pages (the last ``window`` of
    them if given): softmax(scale q.k, capped at ``softcap``) v, f32.  Returns
    out, or (out, lse) with the natural log of the softmax sums; a sequence of
    length 0 gives zeros and -inf.  ``out`` may be q where q is contiguous.
    ``scale`` defaults to 1 / sqrt(head_dim); ``max_len`` (no sequence is
    longer; 0 = what the table holds) sizes the launch and with it the split of
    the sequences, so equal calls give equal bits, but another ``max_len`` may
    change the last ones.  ``ws`` comes from ``paged_attention_workspace``; its
    first word gathers status bits (``read_status``: STATUS_BAD_PAGE for a page
    that does not exist or a length that the table does not hold).  ``status``
    (int32) receives them too, by a small launch of its own, for calls without
    ``ws``."""
    c, dev, seqs, hk, d = _paged_cache(k_cache, v_cache, block_table, k_scale, v_scale)
    shape = q.shape
    if len(shape) != 3:
        raise ValueError("q must be (sequences, q_heads, head_dim)")
    hq = shape[1]
    qs = _rows_f32(q, "q", dev, (seqs, hq, d))
    if out is None:
        out = q.new_empty(seqs, hq, d)
    elif out.dtype is not _F32 or out.get_device() != dev or out.shape != (seqs, hq, d) or \
            not out.is_contiguous():
        _refuse(out, "out", _F32, dev, (seqs, hq, d))
    lse = q.new_empty(seqs, hq) if return_lse else None
    if ws is None:
        ws = paged_attention_workspace(seqs, hq, hk, d, q.device)
    elif ws.dtype is not torch.uint8 or ws.get_device() != dev or not ws.is_contiguous():
        _refuse(ws, "ws", torch.uint8, dev)
    if status is not None:
        _vector(status, _I32, "status", dev, 1)
    _enqueue("moe_paged_attention_record", dev, _ATTENTION_ARGS.pack(
        *c, q.data_ptr(), qs[0], qs[1], _vector(seq_lens, _I32, "seq_lens", dev, seqs),
        out.data_ptr(), 0 if lse is None else lse.data_ptr(), ws.data_ptr(), ws.numel(),
        _raw_stream(dev), hq, max_len, window, d ** -0.5 if scale is None else scale, softcap))
    if status is not None and seqs:
        status |= ws[:4].view(_I32)
    return (out, lse) if return_lse else out


class LinearWeights:
    """A Q4_0 or Q8_0 matrix (rows, cols) for ``linear``: raw GGUF blocks on
    the device, padded to whole tiles and packed once."""

    def __init__(self, raw: torch.Tensor, qtype: int, rows: int, cols: int):
        if qtype not in PACKED_QTYPES:
            raise ValueError(f"unsupported GGML type {qtype} (Q4_0 = 2, Q8_0 = 8)")
        if rows <= 0 or cols <= 0:
            raise ValueError(f"bad shape ({rows}, {cols})")
        _need(raw, torch.uint8, "raw")
        rb = row_bytes(qtype, cols)
        if raw.numel() != rows * rb:
            raise ValueError(f"raw blocks hold {raw.numel()} bytes, expected {rows * rb}")
        self.qtype, self.rows, self.cols, self.device = qtype, rows, cols, raw.device
        pr, pc = -rows % 16, -cols % 64
        if pr or pc:
            raw = torch.nn.functional.pad(raw.view(rows, rb), (0, pc // 32 * BLOCK_BYTES[qtype], 0,
                                                               pr))
        with torch.cuda.device(raw.device):
            self.packed = pack_weights(raw, qtype, 1, rows + pr, cols + pc)
        self.index, self.address = raw.get_device(), self.packed.data_ptr()


def linear(x: torch.Tensor, w: LinearWeights, residual: Optional[torch.Tensor] = None,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x (T, cols) f32 -> (T, rows) f32: W x[t] (+ residual[t]) for a few rows.
    Rows of x, residual and out may stride; out may be residual, but may not
    share memory with x."""
    shape = x.shape
    if len(shape) != 2:
        raise ValueError("x must be (tokens, cols)")
    dev, T = w.index, shape[0]
    xs = _rows_f32(x, "x", dev, (T, w.cols))[0]
    rs = res = 0
    if residual is not None:
        rs, res = _rows_f32(residual, "residual", dev, (T, w.rows))[0], residual.data_ptr()
    if out is None:
        out, ys = x.new_empty(T, w.rows), w.rows
    else:
        ys = _rows_f32(out, "out", dev, (T, w.rows))[0]
        if ys < w.rows and T > 1:
            raise ValueError("rows of out overlap")
    _enqueue("moe_linear_record", dev, _LINEAR_ARGS.pack(
        w.address, x.data_ptr(), xs, res, rs, out.data_ptr(), ys, _raw_stream(dev), w.qtype,
        w.rows, w.cols, T))
    return out


# --------------------------------------------------------------------------- layer

class LayerWeights:
    """Device-resident weights of one MoE layer in the library's layout."""

    def __init__(self, gate_w: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor,
                 w_down: torch.Tensor, qtype: int, E: int, k: int, d: int, F: int,
                 mode: int = 0, bias: Optional[torch.Tensor] = None,
                 router_layout: int = _lib.MOE_ROUTER_D_E,
                 shared: Optional[Tuple[torch.Tensor, torch.Tensor, torch.Tensor]] = None,
                 shared_qtype: int = QTYPE_Q8_0, Fs: int = 0,
                 opts: Optional[ExpertOpts] = None):
        self.gate_w, self.bias = gate_w, bias
        self.opts = opts
        self.w_gate, self.w_up, self.w_down = w_gate, w_up, w_down
        self.shared = shared
        self.qtype, self.E, self.k, self.d, self.F, self.mode = qtype, E, k, d, F, mode
        self.shared_qtype, self.Fs = shared_qtype, Fs
        s = shared or (None, None, None)
        self.c = _lib.MoELayerWeights(
            gate_w.data_ptr(), 0 if bias is None else bias.data_ptr(),
            w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr(),
            0 if s[0] is None else s[0].data_ptr(), 0 if s[1] is None else s[1].data_ptr(),
            0 if s[2] is None else s[2].data_ptr(),
            router_layout, qtype, shared_qtype, E, k, d, F, Fs, mode,
            ctypes.pointer(opts.c) if opts is not None else None)

    def workspace_bytes(self, T: int) -> int:
        out = ctypes.c_size_t(0)
        call("moe_layer_workspace_bytes", ctypes.byref(self.c), T, ctypes.byref(out))
        return int(out.value)


def layer_forward(lw: LayerWeights, x: torch.Tensor, out: Optional[torch.Tensor] = None,
                  residual: Optional[torch.Tensor] = None, ws: Optional[torch.Tensor] = None,
                  ids: Optional[torch.Tensor] = None,
                  weights: Optional[torch.Tensor] = None,
                  router_x: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x and out may be pinned host tensors: the layer then reads x and writes
    out over the bus from its own kernels (no separate copies)."""
    _need(x, torch.float32, "x", pinned_ok=True)
    if out is not None:
        _need(out, torch.float32, "out", pinned_ok=True)
    if router_x is not None:
        _need(router_x, torch.float32, "router_x")
        if router_x.shape != x.shape:
            raise ValueError("router_x must have the shape of x")
    T = x.shape[0]
    if out is None:
        out = torch.empty_like(x) if x.is_cuda else torch.empty(x.shape, dtype=x.dtype,
                                                                 pin_memory=True)
    dev = x.device if x.is_cuda else torch.device("cuda", torch.cuda.current_device())
    if ws is None:
        ws = workspace(lw.workspace_bytes(T), dev)
        ws[:256].zero_()
    call("moe_layer_forward_ex", ctypes.byref(lw.c), _ptr(x), _ptr(router_x), T, _ptr(out),
         _ptr(residual), _ptr(ids), _ptr(weights), _ptr(ws), ws.numel(), _stream())
    return out


def layer_forward_ptr(lw: LayerWeights, x_ptr: int, T: int, out_ptr: int, ws: torch.Tensor,
                      router_x_ptr: int = 0, residual_ptr: int = 0) -> None:
    """moe_layer_forward_ex on raw device pointers (f32 (T, d) rows on the
    current device), for callers that hold their own device buffers."""
    call("moe_layer_forward_ex", ctypes.byref(lw.c), ctypes.c_void_p(int(x_ptr)),
         ctypes.c_void_p(int(router_x_ptr)), T, ctypes.c_void_p(int(out_ptr)),
         ctypes.c_void_p(int(residual_ptr)), None, None, _ptr(ws), ws.numel(), _stream())

"""The attention half of a decode step: a paged key-value cache and the
attention sub-layer over it,

    x + Wo attention(rope(Wq xn), K, V)   with (K, V) += (rope(Wk xn), Wv xn)

for one new token per sequence.  Projections are GGUF Q4_0 / Q8_0 matrices,
rows f32, the cache fp16, bf16 or e4m3.  ``stacked.StackedMoE`` runs it in
front of each MoE layer.
"""
from __future__ import annotations

from typing import List, Optional

import torch

from . import kernels as K
from .moe_forward import Array, _device, _to_dev_u8


class PagedKVCache:
    """Keys and values of up to ``max_seqs`` sequences in pages of
    ``page_size`` tokens, for one layer.  Pages are handed out on the host
    (``reserve`` / ``release``) and listed in ``block_table`` on the device,
    whose address stays the same; a page goes back only with its sequence."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, max_seqs: int,
                 max_pages_per_seq: Optional[int] = None, dtype: torch.dtype = torch.float16,
                 k_scale: float = 1.0, v_scale: float = 1.0, device=None):
        if dtype not in K.CACHE_TYPES:
            raise TypeError(f"caches are {', '.join(str(t) for t in K.CACHE_TYPES)}, not {dtype}")
        if min(pages, page_size, kv_heads, head_dim, max_seqs) <= 0:
            raise ValueError("sizes must be positive")
        dev = _device(device)
        shape = (pages, page_size, kv_heads, head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=dev)
        self.v = torch.zeros(shape, dtype=dtype, device=dev)
        self.k_scale, self.v_scale = float(k_scale), float(v_scale)
        width = min(pages, max_pages_per_seq or pages)
        self.block_table = torch.full((max_seqs, width), -1, dtype=torch.int32, device=dev)
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        self._free: List[int] = list(range(pages - 1, -1, -1))
        self._held: List[List[int]] = [[] for _ in range(max_seqs)]

    @property
    def page_size(self) -> int:
        return self.k.shape[1]

    @property
    def max_seqs(self) -> int:
        return self.block_table.shape[0]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def reserve(self, seq: int, tokens: int) -> None:
        """Makes room for the first ``tokens`` tokens of sequence ``seq``."""
        if not 0 <= seq < self.max_seqs:
            raise IndexError(f"sequence {seq} of {self.max_seqs}")
        held = self._held[seq]
        need = -(-int(tokens) // self.page_size) - len(held)
        if need <= 0:
            return
        if len(held) + need > self.block_table.shape[1]:
            raise ValueError(f"{tokens} tokens need {len(held) + need} pages, a sequence has at "
                             f"most {self.block_table.shape[1]}")
        if need > len(self._free):
            raise RuntimeError(f"cache full: {need} pages needed, {len(self._free)} free")
        new = [self._free.pop() for _ in range(need)]
        at = len(held)
        held += new
        self.block_table[seq, at:at + need] = torch.tensor(new, dtype=torch.int32)

    def release(self, seq: int) -> None:
        """Gives the pages of a finished sequence back."""
        if not 0 <= seq < self.max_seqs:
            raise IndexError(f"sequence {seq} of {self.max_seqs}")
        self._free += reversed(self._held[seq])
        self._held[seq] = []
        self.block_table[seq].fill_(-1)

    def append(self, q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor,
               positions: torch.Tensor, inv_freq: Optional[torch.Tensor] = None,
               seq_ids: Optional[torch.Tensor] = None, interleaved: bool = False,
               q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """``kernels.rope_append`` into this cache."""
        return K.rope_append(q, k, v, self.k, self.v, self.block_table, positions, inv_freq,
                             seq_ids, interleaved, self.k_scale, self.v_scale, q_out, self.status)

    def attend(self, q: torch.Tensor, seq_lens: torch.Tensor, scale: Optional[float] = None,
               window: int = 0, softcap: float = 0.0, max_len: int = 0,
               out: Optional[torch.Tensor] = None, return_lse: bool = False,
               ws: Optional[torch.Tensor] = None):
        """``kernels.paged_attention`` over this cache; q has a row for each
        of the first ``q.shape[0]`` sequences.  Without ``ws`` one is made for
        the call, and its status bits go where the append's do."""
        return K.paged_attention(q, self.k, self.v, self.block_table[:q.shape[0]], seq_lens, scale,
                                 window, softcap, self.k_scale, self.v_scale, max_len, out,
                                 return_lse, ws, self.status if ws is None else None)

    def device_status(self) -> int:
        """Reads and clears the device status bits of the appends and of the
        attention calls without a workspace (synchronises)."""
        st = int(self.status.item())
        self.status.zero_()
        return st


class AttentionLayer:
    """Attention sub-layer of a decode step on GGUF projection matrices: q, k
    and v come from one matrix-vector product of the stacked rows."""

    def __init__(self, w_qkv: K.LinearWeights, w_o: K.LinearWeights, q_heads: int, kv_heads: int,
                 head_dim: int, inv_freq: Optional[torch.Tensor] = None, interleaved: bool = False,
                 window: int = 0, softcap: float = 0.0, scale: Optional[float] = None):
        if q_heads % kv_heads:
            raise ValueError(f"{q_heads} query heads for {kv_heads} key heads")
        if w_qkv.rows != (q_heads + 2 * kv_heads) * head_dim:
            raise ValueError(f"w_qkv has {w_qkv.rows} rows, expected "
                             f"{(q_heads + 2 * kv_heads) * head_dim}")
        if w_o.cols != q_heads * head_dim or w_o.rows != w_qkv.cols:
            raise ValueError(f"w_o is ({w_o.rows}, {w_o.cols}), expected ({w_qkv.cols}, "
                             f"{q_heads * head_dim})")
        self.w_qkv, self.w_o = w_qkv, w_o
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        self.inv_freq, self.interleaved = inv_freq, interleaved
        self.window, self.softcap, self.scale = window, softcap, scale
        self.device = w_qkv.device
        # one workspace for all sizes, cleared here and not in a call that a graph captures
        self._ws = K.paged_attention_workspace(1, q_heads, kv_heads, head_dim, self.device)
        self._qkv, self._att, self._parts = K.RowBuffers(), K.RowBuffers(), {}

    @classmethod
    def from_blocks(cls, w_q: Array, w_k: Array, w_v: Array, w_o: Array, qtype: int, dim: int,
                    q_heads: int, kv_heads: int, head_dim: int, rope_dim: Optional[int] = None,
                    rope_base: float = 10000.0, rope_factors: Optional[torch.Tensor] = None,
                    interleaved: bool = False, window: int = 0, softcap: float = 0.0,
                    scale: Optional[float] = None, device=None) -> "AttentionLayer":
        """From raw block bytes of the ``attn_q`` / ``attn_k`` / ``attn_v`` /
        ``attn_output`` tensors (rows = outputs).  ``rope_dim`` leading
        elements of each head are rotated (default all, 0 none)."""
        dev = _device(device)
        qkv = torch.cat([_to_dev_u8(w, dev) for w in (w_q, w_k, w_v)])
        rope_dim = head_dim if rope_dim is None else rope_dim
        freq = K.rope_inv_freq(rope_dim, rope_base, rope_factors, dev) if rope_dim else None
        return cls(K.LinearWeights(qkv, qtype, (q_heads + 2 * kv_heads) * head_dim, dim),
                   K.LinearWeights(_to_dev_u8(w_o, dev), qtype, dim, q_heads * head_dim),
                   q_heads, kv_heads, head_dim, freq, interleaved, window, softcap, scale)

    def _buffers(self, T: int):
        parts = self._parts.get(T)
        if parts is None:
            hq, hk, d = self.q_heads, self.kv_heads, self.head_dim
            parts = self._parts[T] = (
                self._qkv.rows(T, (hq + 2 * hk) * d, self.device),
                self._att.rows(T, hq * d, self.device).view(T, hq, d), self._ws)
        return parts

    def forward(self, xn: torch.Tensor, cache: PagedKVCache, positions: torch.Tensor,
                seq_lens: torch.Tensor, residual: Optional[torch.Tensor] = None,
                out: Optional[torch.Tensor] = None, max_len: int = 0) -> torch.Tensor:
        """xn (T, dim): the normalised row of the new token of sequences 0 ..
        T - 1, at ``positions`` (int32); ``seq_lens`` counts it (positions + 1
        for a plain decode step; position -1 with length 0 is a padding row).
        ``max_len``: as in ``kernels.paged_attention``; with 0 the launch is sized
        for the longest sequence that the table holds.
        Returns Wo attention (+ residual); ``out`` may be ``residual``.
        Allocates nothing after the first call of a size (but ``out`` when not
        given), and the buffers stay where they are, so captured steps of
        several sizes can be replayed in any order, one after the other."""
        T = xn.shape[0]
        hq, hk, d = self.q_heads, self.kv_heads, self.head_dim
        qkv, att, ws = self._buffers(T)
        K.linear(xn, self.w_qkv, out=qkv)
        q = qkv[:, :hq * d].view(T, hq, d)
        k = qkv[:, hq * d:(hq + hk) * d].view(T, hk, d)
        v = qkv[:, (hq + hk) * d:].view(T, hk, d)
        cache.append(q, k, v, positions, self.inv_freq, None, self.interleaved, q_out=q)
        cache.attend(q, seq_lens, self.scale, self.window, self.softcap, max_len, out=att, ws=ws)
        return K.linear(att.view(T, hq * d), self.w_o, residual=residual, out=out)

    def device_status(self) -> int:
        """Reads and clears the attention's device status bits (synchronises)."""
        return K.read_status(self._ws)

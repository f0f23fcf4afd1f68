"""The attention half of a decode step: a paged key-value cache and the
attention sub-layer over it,

    x + Wo attention(rope(Wq xn), K, V)   with (K, V) += (rope(Wk xn), Wv xn)

for one new token per sequence.  Projections are GGUF Q4_0 / Q8_0 matrices,
rows f32, the cache fp16, bf16 or e4m3; queries and keys may be normed head by
head in front of the rotation.  Sequences may share the pages of a prompt, whose
keys are then read once for all of them, and a cache that keeps account of the
attention its slots receive may be cut down to those that receive most.
``stacked.StackedMoE`` runs the sub-layer in front of each MoE layer.
"""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence

import torch

from . import kernels as K
from .moe_forward import Array, _device, _to_dev_u8


class PagedKVCache:
    """Keys and values of up to ``max_seqs`` sequences in pages of
    ``page_size`` tokens, for one layer.  Pages are handed out on the host
    (``reserve`` / ``trim`` / ``release``) and listed in ``block_table`` on the
    device, whose address stays the same.  Sequences that begin alike may
    ``share`` pages; a page goes back with the last of them.

    With ``track`` the cache has a ledger, ``mass`` and ``held`` (max_seqs,
    kv_heads, slots): the attention that each slot has received (``weigh``) and
    the position of the token in it, by which ``evict`` cuts sequences down.  Its
    slots are ``max_pages_per_seq`` pages for each sequence, 8 bytes each and key
    head: give that number, without it the ledger has room for the whole pool
    ``max_seqs`` times.  An append sets a slot's mass to 0; what a prompt that the
    host appends has received is the host's to write."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, max_seqs: int,
                 max_pages_per_seq: Optional[int] = None, dtype: torch.dtype = torch.float16,
                 k_scale: float = 1.0, v_scale: float = 1.0, device=None, track: bool = False):
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
        self._users = [0] * pages                # sequences of a page
        # lists of shared pages by their last page, while it is in use; then, by length, for others: a
        # captured step may hold their addresses, so their memory is never given back
        self._prefixes: Dict[int, torch.Tensor] = {}
        self._spare: Dict[int, List[torch.Tensor]] = {}
        self._cut = set()                        # sequences that an eviction may have cut down
        self.mass = self.held = None
        if track:
            ledger = (max_seqs, kv_heads, width * page_size)
            self.mass = torch.zeros(ledger, dtype=torch.float32, device=dev)
            self.held = torch.full(ledger, -1, dtype=torch.int32, device=dev)

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
        for page in new:
            self._users[page] = 1
        self._list(seq, new)

    def _list(self, seq: int, pages: List[int]) -> None:
        held = self._held[seq]
        at = len(held)
        held += pages
        self.block_table[seq, at:at + len(pages)] = torch.tensor(pages, dtype=torch.int32)

    def trim(self, seq: int, tokens: int) -> None:
        """Gives the pages behind the first ``tokens`` tokens (slots) of a sequence back."""
        if not 0 <= seq < self.max_seqs:
            raise IndexError(f"sequence {seq} of {self.max_seqs}")
        keep = -(-max(int(tokens), 0) // self.page_size)
        if keep == 0:
            self._cut.discard(seq)
        gone = self._held[seq][keep:]
        if not gone:
            return
        del self._held[seq][keep:]
        for page in reversed(gone):
            self._users[page] -= 1
            if not self._users[page]:
                self._free.append(page)
                pages = self._prefixes.pop(page, None)
                if pages is not None:
                    self._spare.setdefault(pages.numel(), []).append(pages)
        self.block_table[seq, keep:] = -1

    def release(self, seq: int) -> None:
        """Gives the pages of a finished sequence back."""
        self.trim(seq, 0)

    def share(self, seq: int, other: int, tokens: int) -> None:
        """Lets ``seq``, which holds nothing, begin with the pages of the first
        ``tokens`` tokens of sequence ``other`` (whole pages).  Neither may write
        to them any more; what follows them is ``seq``'s own."""
        for s in (seq, other):
            if not 0 <= s < self.max_seqs:
                raise IndexError(f"sequence {s} of {self.max_seqs}")
        if self.mass is not None:
            raise ValueError("a cache that evicts shares no pages")
        if tokens < 0 or tokens % self.page_size:
            raise ValueError(f"{tokens} tokens are not whole pages of {self.page_size}")
        n = tokens // self.page_size
        if self._held[seq] or n > len(self._held[other]):
            raise ValueError(f"sequence {seq} holds {len(self._held[seq])} pages, sequence {other} "
                             f"{len(self._held[other])}: none, and {n}, are needed")
        pages = self._held[other][:n]
        for page in pages:
            self._users[page] += 1
        if pages:
            self._list(seq, pages)

    def prefix(self, seq: int, tokens: int) -> torch.Tensor:
        """The pages of the first ``tokens`` tokens (whole pages, which it holds) of a
        sequence, for ``attend``.  A list of its own, not part of the block table: it stays
        right for the sequences that share these pages when this one is released or
        trimmed, and a captured step may be replayed for them.  It is made at the first
        call, which can not be captured; later calls return the same tensor.  When the
        last sequence has given the pages back it may become another prompt's list."""
        if not 0 <= seq < self.max_seqs:
            raise IndexError(f"sequence {seq} of {self.max_seqs}")
        n = tokens // self.page_size
        if tokens < 0 or tokens % self.page_size or n > self.block_table.shape[1]:
            raise ValueError(f"{tokens} tokens are not whole pages of {self.page_size} of a sequence")
        held = self._held[seq]
        if n > len(held):
            raise ValueError(f"sequence {seq} holds {len(held)} pages, {n} are needed")
        if n == 0:
            return self.block_table[seq, :0]
        # A page that several sequences hold came to them with all pages in front of it, and
        # those can not change while they hold it: the last page tells the list
        pages = self._prefixes.get(held[n - 1])
        if pages is None:
            if self.block_table.is_cuda and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("call prefix() once before a capture")
            pages = torch.tensor(held[:n], dtype=torch.int32, device=self.block_table.device)
            if self._spare.get(n):
                pages = self._spare[n].pop().copy_(pages)
            self._prefixes[held[n - 1]] = pages
        return pages

    def append(self, q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor,
               positions: torch.Tensor, inv_freq: Optional[torch.Tensor] = None,
               seq_ids: Optional[torch.Tensor] = None, interleaved: bool = False,
               q_out: Optional[torch.Tensor] = None, q_norm: Optional[torch.Tensor] = None,
               k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6,
               gemma_style: bool = False,
               slots: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """``kernels.rope_append`` into this cache and its ledger.  ``slots``
        (default: the positions) where an eviction has set them apart."""
        return K.rope_append(q, k, v, self.k, self.v, self.block_table, positions, inv_freq,
                             seq_ids, interleaved, self.k_scale, self.v_scale, q_out, self.status,
                             q_norm, k_norm, eps, gemma_style, slots, self.mass, self.held)

    def check_window(self, window: int, seqs: int, prefix: Optional[torch.Tensor] = None) -> None:
        """Refuses a window over the first ``seqs`` sequences where it would not be the newest
        tokens: behind an eviction those sit in any slots, until the sequence is released."""
        if window and prefix is not None:
            raise ValueError("a window does not go with a shared prefix")
        if window and self._cut and min(self._cut) < seqs:
            raise ValueError(f"a window does not go with an eviction: sequence {min(self._cut)} has "
                             "been cut down, its slots are not in the order of its tokens")

    def attend(self, q: torch.Tensor, seq_lens: torch.Tensor, scale: Optional[float] = None,
               window: int = 0, softcap: float = 0.0, max_len: int = 0,
               out: Optional[torch.Tensor] = None, return_lse: bool = False,
               ws: Optional[torch.Tensor] = None, prefix: Optional[torch.Tensor] = None,
               lse_out: Optional[torch.Tensor] = None):
        """``kernels.paged_attention`` over this cache; q has a row for each
        of the first ``q.shape[0]`` sequences.  Without ``ws`` one is made for
        the call, and its status bits go where the append's do.  ``prefix``: the
        pages that all of these sequences begin with (``kernels.prefix_attention``
        and its workspace; no window)."""
        self.check_window(window, q.shape[0], prefix)
        table, status = self.block_table[:q.shape[0]], self.status if ws is None else None
        if prefix is None:
            return K.paged_attention(q, self.k, self.v, table, seq_lens, scale, window, softcap,
                                     self.k_scale, self.v_scale, max_len, out, return_lse, ws,
                                     status, lse_out)
        return K.prefix_attention(q, self.k, self.v, table, seq_lens, prefix, scale, softcap,
                                  self.k_scale, self.v_scale, max_len, out, return_lse, ws, status,
                                  lse_out=lse_out)

    def weigh(self, q: torch.Tensor, seq_lens: torch.Tensor, lse: torch.Tensor,
              scale: Optional[float] = None, window: int = 0, softcap: float = 0.0,
              max_len: int = 0) -> None:
        """Adds the attention of ``attend`` with the same arguments, which returned
        ``lse``, to the ledger (``kernels.attention_mass``)."""
        if self.mass is None:
            raise ValueError("the cache keeps no ledger (track=True)")
        S = q.shape[0]
        self.check_window(window, S)
        K.attention_mass(q, self.k, self.block_table[:S], seq_lens, lse, self.mass[:S], scale, window,
                         softcap, self.k_scale, max_len, status=self.status)

    def evict(self, seq_lens: torch.Tensor, keep: int, recent: int = 0, max_len: int = 0,
              lens_out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Cuts the first ``len(seq_lens)`` sequences down to ``keep`` slots each
        (``kernels.cache_evict``), in place; ``lens_out`` (default: seq_lens itself)
        receives the new lengths.  ``max_len``, which no sequence exceeds, picks the kernel:
        ``keep + 1`` where each step gives up one slot.  ``trim`` then gives their pages
        back.  Layers that share seq_lens: see ``evict``.  Windows over a sequence are
        refused from then on, until it is released."""
        if self.mass is None:
            raise ValueError("the cache keeps no ledger (track=True)")
        S = seq_lens.shape[0]
        lens = K.cache_evict(self.k, self.v, self.block_table[:S], seq_lens, self.mass[:S],
                             self.held[:S], keep, recent, lens_out=lens_out, max_len=max_len,
                             status=self.status)
        self._cut.update(range(S))
        return lens

    def device_status(self) -> int:
        """Reads and clears the device status bits of the appends, of the ledger
        and of the attention calls without a workspace (synchronises)."""
        st = int(self.status.item())
        self.status.zero_()
        return st


def evict(caches: Sequence[PagedKVCache], seq_lens: torch.Tensor, keep: int, recent: int = 0,
          max_len: int = 0) -> torch.Tensor:
    """``PagedKVCache.evict`` in the caches of all layers, which share seq_lens: each
    layer keeps slots of its own choice, and the lengths change once, at the end.
    ``max_len``: ``keep + 1`` where each step gives up one slot."""
    others = torch.empty_like(seq_lens)
    for cache in caches[:-1]:
        cache.evict(seq_lens, keep, recent, max_len, others)
    if caches:
        caches[-1].evict(seq_lens, keep, recent, max_len)
    return seq_lens


class AttentionLayer:
    """Attention sub-layer of a decode step on GGUF projection matrices: q, k
    and v come from one matrix-vector product of the stacked rows."""

    def __init__(self, w_qkv: K.LinearWeights, w_o: K.LinearWeights, q_heads: int, kv_heads: int,
                 head_dim: int, inv_freq: Optional[torch.Tensor] = None, interleaved: bool = False,
                 window: int = 0, softcap: float = 0.0, scale: Optional[float] = None,
                 q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None,
                 norm_eps: float = 1e-6, gemma_style: bool = False):
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
        self.q_norm, self.k_norm, self.norm_eps = q_norm, k_norm, norm_eps
        self.gemma_style = gemma_style
        self.device = w_qkv.device
        # one workspace for all sizes, cleared here and not in a call that a graph captures
        self._ws = K.paged_attention_workspace(1, q_heads, kv_heads, head_dim, self.device)
        self._qkv, self._att, self._parts = K.RowBuffers(), K.RowBuffers(), {}
        self._lse, self._prefix_ws = K.RowBuffers(), {}

    @classmethod
    def from_blocks(cls, w_q: Array, w_k: Array, w_v: Array, w_o: Array, qtype: int, dim: int,
                    q_heads: int, kv_heads: int, head_dim: int, rope_dim: Optional[int] = None,
                    rope_base: float = 10000.0, rope_factors: Optional[torch.Tensor] = None,
                    interleaved: bool = False, window: int = 0, softcap: float = 0.0,
                    scale: Optional[float] = None, device=None,
                    q_norm: Optional[Array] = None, k_norm: Optional[Array] = None,
                    norm_eps: float = 1e-6, gemma_style: bool = False) -> "AttentionLayer":
        """From raw block bytes of the ``attn_q`` / ``attn_k`` / ``attn_v`` /
        ``attn_output`` tensors (rows = outputs).  ``rope_dim`` leading
        elements of each head are rotated (default all, 0 none).  ``q_norm``,
        ``k_norm`` (head_dim,): the ``attn_q_norm`` / ``attn_k_norm`` weights of
        models that norm each head."""
        dev = _device(device)
        qkv = torch.cat([_to_dev_u8(w, dev) for w in (w_q, w_k, w_v)])
        rope_dim = head_dim if rope_dim is None else rope_dim
        freq = K.rope_inv_freq(rope_dim, rope_base, rope_factors, dev) if rope_dim else None
        return cls(K.LinearWeights(qkv, qtype, (q_heads + 2 * kv_heads) * head_dim, dim),
                   K.LinearWeights(_to_dev_u8(w_o, dev), qtype, dim, q_heads * head_dim),
                   q_heads, kv_heads, head_dim, freq, interleaved, window, softcap, scale,
                   *(None if w is None else torch.as_tensor(w).to(dev, torch.float32).contiguous()
                     for w in (q_norm, k_norm)), norm_eps, gemma_style)

    def _buffers(self, T: int):
        parts = self._parts.get(T)
        if parts is None:
            hq, hk, d = self.q_heads, self.kv_heads, self.head_dim
            parts = self._parts[T] = (
                self._qkv.rows(T, (hq + 2 * hk) * d, self.device),
                self._att.rows(T, hq * d, self.device).view(T, hq, d), self._ws)
        return parts

    def _prefix_workspace(self, T: int) -> Optional[torch.Tensor]:
        """As the row buffers: one for each power of two of rows, never replaced.  None
        where it would have to be made in a capture: it would be cleared when the
        graph is replayed, but not before a call that is not part of the graph (then
        one is made for the captured call alone, with its status in the cache's)."""
        rows = 1 << max(T - 1, 0).bit_length()
        ws = self._prefix_ws.get(rows)
        if ws is None and not torch.cuda.is_current_stream_capturing():
            ws = self._prefix_ws[rows] = K.prefix_attention_workspace(
                rows, self.q_heads, self.kv_heads, self.head_dim, self.device)
        return ws

    def check_step(self, seqs: int, cache: PagedKVCache, prefix: Optional[torch.Tensor] = None,
                   slots: Optional[torch.Tensor] = None) -> None:
        """Refuses what ``forward`` can not take together, before anything is written."""
        if self.window and slots is not None:
            raise ValueError("a window counts slots and does not go with slots apart from the "
                             "positions")
        cache.check_window(self.window, seqs, prefix)

    def forward(self, xn: torch.Tensor, cache: PagedKVCache, positions: torch.Tensor,
                seq_lens: torch.Tensor, residual: Optional[torch.Tensor] = None,
                out: Optional[torch.Tensor] = None, max_len: int = 0,
                prefix: Optional[torch.Tensor] = None,
                slots: Optional[torch.Tensor] = None) -> torch.Tensor:
        """xn (T, dim): the normalised row of the new token of sequences 0 ..
        T - 1, at ``positions`` (int32); ``seq_lens`` counts it (positions + 1
        for a plain decode step; position -1 with length 0 is a padding row).
        ``max_len``: as in ``kernels.paged_attention``; with 0 the launch is sized
        for the longest sequence that the table holds.
        ``prefix``: the pages that all of these sequences begin with
        (``PagedKVCache.prefix``).  ``slots`` (int32): where the new tokens go, if
        that is not their positions (behind an eviction seq_lens - 1).  A layer with a
        window takes neither.  A cache with a ledger receives the step's attention.
        Returns Wo attention (+ residual); ``out`` may be ``residual``.
        Allocates nothing after the first call of a size (but ``out`` when not
        given), and the buffers stay where they are, so captured steps of
        several sizes can be replayed in any order, one after the other."""
        T = xn.shape[0]
        self.check_step(T, cache, prefix, slots)
        hq, hk, d = self.q_heads, self.kv_heads, self.head_dim
        qkv, att, ws = self._buffers(T)
        K.linear(xn, self.w_qkv, out=qkv)
        q = qkv[:, :hq * d].view(T, hq, d)
        k = qkv[:, hq * d:(hq + hk) * d].view(T, hk, d)
        v = qkv[:, (hq + hk) * d:].view(T, hk, d)
        cache.append(q, k, v, positions, self.inv_freq, None, self.interleaved, q, self.q_norm,
                     self.k_norm, self.norm_eps, self.gemma_style, slots)
        lse = None if cache.mass is None else self._lse.rows(T, hq, self.device)
        if prefix is not None:
            ws = self._prefix_workspace(T)
        cache.attend(q, seq_lens, self.scale, self.window, self.softcap, max_len, out=att, ws=ws,
                     prefix=prefix, lse_out=lse)
        if lse is not None:
            cache.weigh(q, seq_lens, lse, self.scale, self.window, self.softcap, max_len)
        return K.linear(att.view(T, hq * d), self.w_o, residual=residual, out=out)

    def device_status(self) -> int:
        """Reads and clears the attention's device status bits (synchronises)."""
        st = K.read_status(self._ws)
        for ws in self._prefix_ws.values():
            st |= K.read_status(ws)
        return st

"""Stacked decode step: L MoE layers, each with an always-on shared expert,
with the residual and RMSNorm of MoETransformerModel._layer_forward
(moe_forward.py:348-359): ``x = x + moe(rms_norm(x, w))``, after ``x = x +
attention(rms_norm(x, wa))`` where the stack has attention layers."""
from __future__ import annotations

from typing import List, Optional, Sequence

import torch

from . import kernels as K
from .attention import AttentionLayer, PagedKVCache
from .moe_forward import MoELayer


class StackedMoE:
    """``attention`` (an ``AttentionLayer`` per MoE layer) with
    ``attention_norms`` makes whole decoder layers of the stack."""

    def __init__(self, layers: Sequence[MoELayer], norms: Sequence[torch.Tensor], eps: float = 1e-6,
                 attention: Optional[Sequence[AttentionLayer]] = None,
                 attention_norms: Optional[Sequence[torch.Tensor]] = None):
        self.layers = list(layers)
        self.norms = list(norms)
        self.eps = eps
        self.attention = list(attention) if attention is not None else None
        self.attention_norms = list(attention_norms) if attention_norms is not None else None
        if (self.attention is None) != (self.attention_norms is None):
            raise ValueError("attention and attention_norms come together")
        if self.attention is not None and not (
                len(self.attention) == len(self.attention_norms) == len(self.layers)):
            raise ValueError(f"{len(self.attention)} attention layers and "
                             f"{len(self.attention_norms)} norms for {len(self.layers)} MoE layers")
        self._xn = K.RowBuffers()

    @classmethod
    def from_layers(cls, datas, device=None, eps: float = 1e-6) -> "StackedMoE":
        """From synthetic layer data (``synth.MoELayerData`` per layer)."""
        layers, norms = [], []
        for data in datas:
            cfg = data.cfg
            shared = None
            if cfg.shared_ffn:
                shared = (data.s_gate[0], data.s_up[0], data.s_down[0])
            layer = MoELayer.from_blocks(data.gate_w, data.w_gate, data.w_up, data.w_down,
                                         cfg.qtype, cfg.top_k, shared=shared,
                                         shared_qtype=cfg.shared_qtype,
                                         shared_hidden=cfg.shared_ffn, bias=data.bias,
                                         device=device)
            layers.append(layer)
            norms.append(torch.from_numpy(data.norm_w).to(layer.router.device))
        return cls(layers, norms, eps)

    def forward(self, x: torch.Tensor, out: Optional[torch.Tensor] = None,
                caches: Optional[Sequence[PagedKVCache]] = None,
                positions: Optional[torch.Tensor] = None,
                seq_lens: Optional[torch.Tensor] = None, max_len: int = 0) -> torch.Tensor:
        """x (T, d) f32 on the device -> (T, d).  The residual stream lives in
        ``out`` (allocated if not given): the first layer adds x into it,
        later layers update it in place (the combine may write over its own
        residual input), so a step with ``out`` allocates nothing after
        the first of its size.

        With attention layers row t is the new token of sequence t:
        ``caches`` (one per layer), ``positions`` and ``seq_lens`` as
        ``AttentionLayer.forward`` takes them."""
        if self.attention is not None:
            if caches is None or positions is None or seq_lens is None:
                raise ValueError("attention layers need caches, positions and seq_lens")
            if len(caches) != len(self.layers):
                raise ValueError(f"{len(caches)} caches for {len(self.layers)} layers")
        xn = self._xn.rows(*x.shape, x.device)
        res = out if out is not None else torch.empty_like(x)
        cur = x
        for i, (layer, nw) in enumerate(zip(self.layers, self.norms)):
            if self.attention is not None:
                K.rms_norm(cur, self.attention_norms[i], self.eps, out=xn)
                self.attention[i].forward(xn, caches[i], positions, seq_lens, residual=cur,
                                          out=res, max_len=max_len)
                cur = res
            K.rms_norm(cur, nw, self.eps, out=xn)
            layer.forward_batch(xn, residual=cur, out=res)
            cur = res
        return res


class StackedEP:
    """The stacked step with every layer expert-parallel over ``group``: the
    layers share one exchange window; RMSNorm and the residual are local."""

    def __init__(self, layers, norms, eps: float = 1e-6):
        self.layers = list(layers)
        self.norms = list(norms)
        self.eps = eps
        self._xn = K.RowBuffers()

    @classmethod
    def build(cls, cfg, seed: int, tokens: int, group=None, device=None, eps: float = 1e-6,
              layers: Optional[int] = None) -> "StackedEP":
        """Synthetic layers (seed + layer index); each rank generates and packs
        only its own experts."""
        import torch.distributed as dist
        from . import synth
        from .ep import EPExchange, EPMoELayer, expert_range
        rank, world = dist.get_rank(group), dist.get_world_size(group)
        e0, e1 = expert_range(rank, world, cfg.n_experts)
        ex = EPExchange(group, device)
        ls, ns = [], []
        for li in range(cfg.n_layers if layers is None else layers):
            data = synth.make_layer_slice(cfg, seed + li, tokens * world, e0, e1)
            shared = (data.s_gate, data.s_up, data.s_down) if cfg.shared_ffn else None
            layer = EPMoELayer(data.gate_w, data.w_gate, data.w_up, data.w_down, cfg.qtype,
                               cfg.top_k, cfg.route_mode, None, group=group, device=device,
                               shared=shared, shared_qtype=cfg.shared_qtype, local=True,
                               exchange=ex)
            ls.append(layer)
            ns.append(torch.from_numpy(data.norm_w).to(layer.device))
        return cls(ls, ns, eps)

    @classmethod
    def from_layers(cls, datas, group=None, device=None, eps: float = 1e-6) -> "StackedEP":
        """From per-layer data whose expert stacks hold this rank's experts
        only (``synth.make_layer_device`` / ``make_layer_slice`` for the rank's
        expert range); the layers share one exchange window."""
        from .ep import EPExchange, EPMoELayer
        ex = EPExchange(group, device)
        ls, ns = [], []
        for data in datas:
            cfg = data.cfg
            shared = (data.s_gate, data.s_up, data.s_down) if cfg.shared_ffn else None
            layer = EPMoELayer(data.gate_w, data.w_gate, data.w_up, data.w_down, cfg.qtype,
                               cfg.top_k, cfg.route_mode, data.bias, group=group, device=device,
                               shared=shared, shared_qtype=cfg.shared_qtype, local=True,
                               exchange=ex)
            ls.append(layer)
            ns.append(torch.from_numpy(data.norm_w).to(layer.device))
        return cls(ls, ns, eps)

    def close(self) -> None:
        if self.layers:
            self.layers[0].exchange.close()

    def forward(self, x: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """As ``StackedMoE.forward``, every layer expert-parallel."""
        xn = self._xn.rows(*x.shape, x.device)
        res = out if out is not None else torch.empty_like(x)
        cur = x
        for layer, nw in zip(self.layers, self.norms):
            K.rms_norm(cur, nw, self.eps, out=xn)
            layer.forward(xn, out=res, residual=cur)
            cur = res
        return res

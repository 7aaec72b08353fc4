"""The half of a decoder layer behind its attention, from 4-bit weights: dense or a mixture of experts.

    layer = DecoderLayer(AttentionBlock(..., norm=w1), MLPBlock(gate_up, down, norm=w2))
    layer = DecoderLayer(AttentionBlock(..., norm=w1), ExpertBlock(router, gate_up, down, k, norm=w2))

A block takes the residual stream x (fp16 [tokens, hidden]) and returns it with its own result added: the norm, the gated
product and the product back are ``rms_norm``, ``w4a16_linear`` or ``moe_route`` and ``moe_experts``; a layer is called
as an attention block is, and ``attention_block.DecodeLoop`` runs its single-token steps from a captured graph.
"""
from __future__ import annotations

import torch

from .attention_block import AttentionBlock
from .layer import rms_norm, w4a16_linear
from .moe import moe_experts, moe_route


class MLPBlock:
    """x + down(act(gate(norm x)) * up(norm x)); ``gate_up`` and ``down`` are (packed words, scales), the first's rows
    laid by ``interleave_gate_up``."""

    def __init__(self, gate_up, down, norm: torch.Tensor, eps: float = 1e-5, activation: str = "silu"):
        self.gate_up, self.down, self.norm, self.eps, self.activation = gate_up, down, norm, eps, activation

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        h = rms_norm(x, self.norm, self.eps)
        h = w4a16_linear(self.gate_up[0], h, self.gate_up[1], activation=self.activation, gated=True)
        return w4a16_linear(self.down[0], h, self.down[1], residual=x)


class ExpertBlock:
    """x + the weighted sum of each token's ``k`` experts over norm x.  ``router`` is fp16 [hidden, experts] (its product a
    plain 16-bit one); ``gate_up`` and ``down`` as ``moe_experts`` takes them."""

    def __init__(self, router: torch.Tensor, gate_up, down, k: int, norm: torch.Tensor, eps: float = 1e-5,
                 activation: str = "silu", renormalize: bool = True):
        self.router, self.gate_up, self.down, self.k, self.norm = router, gate_up, down, k, norm
        self.eps, self.activation, self.renormalize = eps, activation, renormalize

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        h = rms_norm(x, self.norm, self.eps)
        weights, experts = moe_route(h @ self.router, self.k, renormalize=self.renormalize)
        return moe_experts(h, self.gate_up, self.down, experts, weights, activation=self.activation, residual=x)


class DecoderLayer:
    """An attention block with its norm, then ``mlp`` (either block above), on the residual stream."""

    def __init__(self, attention: AttentionBlock, mlp):
        if attention.norm is None:
            raise RuntimeError("a layer's attention block needs its norm: without one it does not add to the residual stream")
        self.attention, self.mlp = attention, mlp

    @property
    def cache(self):
        return self.attention.cache

    def __call__(self, x, positions, slots, page_table, seq_lens, **kwargs):
        return self.mlp(self.attention(x, positions, slots, page_table, seq_lens, **kwargs))

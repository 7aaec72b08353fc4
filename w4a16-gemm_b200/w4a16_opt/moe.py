"""A mixture of experts from 4-bit weights: its router, its experts.

    weights, experts = moe_route(h @ router, k)
    x = moe_experts(h, gate_up, down, experts, weights, residual=x, out=x)

The reference has no counterpart.  Every function runs on the current CUDA stream, and raises
RuntimeError on bad input.
"""
from __future__ import annotations

import torch

from . import _C
from .layer import activation_code


def moe_route(logits: torch.Tensor, k: int, *, renormalize: bool = True):
    """The ``k`` experts of largest softmax weight for each token: (weights fp32, experts int32), both [tokens, k].

    ``logits`` [tokens, experts], fp16, bf16 or fp32, last dimension dense, at most 1024 experts; k at most 32.
    Experts come in falling order of their logits, equal ones by index.  Weights are those of the softmax over all
    experts, divided by their sum with ``renormalize``.  A logit of -inf or NaN is never chosen; where fewer than k are
    left, the rest of the row is expert -1 with weight 0.
    """
    return _C.moe_route(logits, k, renormalize)


def moe_experts(x: torch.Tensor, gate_up, down, experts: torch.Tensor, weights: torch.Tensor, *,
                activation: str | None = "silu", residual: torch.Tensor | None = None, out: torch.Tensor | None = None,
                workspace: torch.Tensor | None = None) -> torch.Tensor:
    """y_t = residual_t + sum_j weights[t, j] * down_e(act(gate_e(x_t)) * up_e(x_t)), e = experts[t, j]; fp16 [tokens, hidden].

    ``x`` fp16 [tokens, hidden].  ``gate_up`` and ``down`` are (packed words, scales) of all experts, stacked: int32
    [experts, 2 * inner * hidden / 8] and fp16 [experts, hidden/G, 2 * inner], rows laid by ``interleave_gate_up``;
    int32 [experts, hidden * inner / 8] and fp16 [experts, inner/G, hidden].  hidden and inner are multiples of 64 and of their
    group size (64 or 128); at most 1024 experts.  ``experts`` int32 and ``weights`` fp32 [tokens, k], as ``moe_route``
    gives them; an expert outside [0, experts) adds nothing (another device's, say), the same one twice counts twice.

    Sums are fp32; the inner results act(gate) * up are rounded to fp16, as ``w4a16_linear`` would return them, and y once: where
    an inner result passes fp16's 65504, its token's y is not finite.  For a given number of tokens a token's y depends on
    its own inputs alone, bit for bit.  tokens * k * max(inner / 8, hidden / 4) must be below 2^31.

    ``out`` may be ``residual`` or ``x``.  ``workspace``: optional scratch CUDA buffer (256-byte aligned); without it the binding
    keeps one per (device, stream) for calls that need up to 64 MB, and takes a larger one from torch's allocator for the call.
    """
    return _C.moe_experts(x, gate_up[0], gate_up[1], down[0], down[1], experts, weights, activation_code(activation),
                          residual, out, workspace)

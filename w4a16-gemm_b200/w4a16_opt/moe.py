"""A mixture of experts: its router.

    weights, experts = moe_route(logits, k)

The reference has no counterpart.  Every function runs on the current CUDA stream, and raises
RuntimeError on bad input.
"""
from __future__ import annotations

import torch

from . import _C


def moe_route(logits: torch.Tensor, k: int, *, renormalize: bool = True):
    """The ``k`` experts of largest softmax weight for each token: (weights fp32, experts int32), both [tokens, k].

    ``logits`` [tokens, experts], fp16, bf16 or fp32, last dimension dense, at most 1024 experts; k at most 32.
    Experts come in falling order of their logits, equal ones by index.  Weights are those of the softmax over all
    experts, divided by their sum with ``renormalize``.  A logit of -inf or NaN is never chosen; where fewer than k are
    left, the rest of the row is expert -1 with weight 0.
    """
    return _C.moe_route(logits, k, renormalize)

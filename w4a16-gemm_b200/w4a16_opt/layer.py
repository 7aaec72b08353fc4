"""What stands around the products of a decoder layer: a product with its epilogue, the norm before it.

    h, x = rms_norm(y, weight, residual=x)                               # x += y; h = norm(x)
    h = w4a16_linear(Wgu, h, sgu, activation="silu", gated=True)         # silu(h Wg^T) * (h Wu^T)
    x = w4a16_linear(Wd, h, sd, residual=x, out=x)                       # x += h Wd^T

The reference has the product alone.  Every function runs on the current CUDA stream, and raises
RuntimeError on bad input.
"""
from __future__ import annotations

import torch

from . import _C

ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}


def activation_code(activation) -> int:
    if activation not in ACTIVATIONS:
        raise RuntimeError(f"activation must be one of {[a for a in ACTIVATIONS if a]}, not {activation!r}")
    return ACTIVATIONS[activation]


def interleave_gate_up(gate: torch.Tensor, up: torch.Tensor, dim: int = 0) -> torch.Tensor:
    """The rows (of dimension ``dim``) of a gated weight: eight of ``gate``, eight of ``up``, eight of ``gate``, ...

    For weights before ``quantize_pack``, codes before ``pack_int4`` (``dim=0``), scales [K/G, N] (``dim=1``) and
    biases.  That dimension must be a multiple of 8.
    """
    if gate.shape != up.shape:
        raise RuntimeError("gate and up must have one shape")
    if gate.shape[dim] % 8:
        raise RuntimeError("a gated weight must have a multiple of 8 rows for each factor")
    dim %= gate.dim()
    both = torch.stack((gate.unflatten(dim, (-1, 8)), up.unflatten(dim, (-1, 8))), dim + 1)
    return both.flatten(dim, dim + 2)


def w4a16_linear(Wp: torch.Tensor, x: torch.Tensor, scales: torch.Tensor, *, bias: torch.Tensor | None = None,
                 activation: str | None = None, gated: bool = False, residual: torch.Tensor | None = None,
                 out: torch.Tensor | None = None, variant: int = -1, workspace: torch.Tensor | None = None,
                 weights_resident: bool = False, fp32_scale: bool = False) -> torch.Tensor:
    """``w4a16_gemm`` with an epilogue: act(x W^T + bias) + residual, rounded to fp16 once.

    ``activation``: None, "relu", "silu", "gelu" (by the normal distribution) or "gelu_tanh".  ``bias`` fp16 [N].
    ``gated``: the weight's rows (and bias) alternate as ``interleave_gate_up`` lays them, and y[:, j] = act(gate_j) *
    up_j + residual, N / 2 columns.  ``residual`` fp16 of y's shape; ``out``, where y goes, may be the residual
    itself, and must not overlap anything else that is read.  The other arguments are those of ``w4a16_gemm_out``, and so
    are the products: with nothing but a product asked for, the result is ``w4a16_gemm``'s bit for bit.
    """
    return _C.linear(Wp, x, scales, bias, activation_code(activation), gated, residual, out, variant, workspace,
                     weights_resident, fp32_scale)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, *, residual: torch.Tensor | None = None,
             out: torch.Tensor | None = None, residual_out: torch.Tensor | None = None):
    """x * weight / sqrt(mean(x^2) + eps) over the last dimension; with ``residual``, (that of x + residual, x + residual).

    ``x`` fp16 or bf16 [dim], [tokens, dim] or [tokens, heads, dim] (heads of a fused projection, say) with a dense
    last dimension, other strides multiples of 8; dim a multiple of 8 up to 32768.  ``weight`` [dim] of x's dtype.
    ``residual`` of x's shape, in x's dtype or fp32; the sum is returned in its type, and the norm
    taken of the unrounded sum.  ``out`` and ``residual_out``, where the results go, may be ``x`` or ``residual``
    themselves (the very same view) and otherwise lie apart from every input, from first address to last (views that alternate in
    one buffer are refused).
    """
    y, h = _C.rms_norm(x, weight, eps, residual, out, residual_out)
    return y if residual is None else (y, h)

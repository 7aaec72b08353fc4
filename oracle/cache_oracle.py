"""Plain 64-bit restatement of the 4-bit key/value cache and of attention over it.

Written from the definitions only: nothing here calls the package.  Works on torch tensors of any
device; every computed number is fp64.
"""
from __future__ import annotations

import math

import torch

LIMIT = 57344.0


def block_bytes(page_size, head_dim, group_size):
    return page_size * (head_dim + 8 * (head_dim // group_size))


def quantise(x, group_size):
    """fp64 values [..., D] -> (codes uint8 [..., D], scales fp16, minima fp16 [..., D / G])."""
    x = x.double().nan_to_num(nan=0.0, posinf=LIMIT, neginf=-LIMIT).clamp(-LIMIT, LIMIT)
    g = x.reshape(*x.shape[:-1], x.shape[-1] // group_size, group_size)
    low = g.amin(-1).half()
    # the scale is a quotient in fp32, then fp16
    step = ((g.amax(-1).float() - low.float()).clamp(min=0) / torch.full((), 15.0, device=x.device)).half()
    s = step.double().unsqueeze(-1)
    code = torch.where(s > 0, ((g - low.double().unsqueeze(-1)) / torch.where(s > 0, s, 1.0)).round(), 0.0)
    return code.clamp(0, 15).to(torch.uint8).reshape(x.shape), step, low


def values(codes, scales, minima, group_size):
    g = codes.double().reshape(*codes.shape[:-1], codes.shape[-1] // group_size, group_size)
    return (g * scales.double().unsqueeze(-1) + minima.double().unsqueeze(-1)).reshape(codes.shape)


def write_block(block, page_size, row, key, value):
    """Puts one token's (codes, scales, minima) of key and value into a block (uint8 [bytes])."""
    d = key[0].numel()
    ng = key[1].numel()
    for which, (codes, scales, minima) in enumerate((key, value)):
        packed = codes[0::2] | (codes[1::2] << 4)
        at = which * page_size * d // 2 + row * d // 2
        block[at:at + d // 2] = packed
        pairs = torch.stack((scales, minima), -1).reshape(-1).contiguous().view(torch.uint8)
        at = page_size * d + which * page_size * 4 * ng + row * 4 * ng
        block[at:at + 4 * ng] = pairs


def read_slots(data, head_dim, page_size, group_size, slots):
    """fp64 keys and values [tokens, heads, D] of a cache's slots."""
    pages, heads, _ = data.shape
    ng, n = head_dim // group_size, page_size * head_dim // 2
    flat = data.reshape(pages, heads, -1)
    out = []
    for which in (0, 1):
        c = flat[:, :, which * n:(which + 1) * n].reshape(pages, heads, page_size, head_dim // 2)
        c = c[slots // page_size, :, slots % page_size]
        codes = torch.stack((c & 15, c >> 4), -1).flatten(-2)
        at = 2 * n + which * page_size * 4 * ng
        p = flat[:, :, at:at + page_size * 4 * ng].contiguous().view(torch.float16)
        p = p.reshape(pages, heads, page_size, ng, 2)[slots // page_size, :, slots % page_size]
        out.append(values(codes, p[..., 0], p[..., 1], group_size))
    return out


def rotate(x, positions, cos_sin, sections=None, interleaved=False):
    """x [T, heads, D] fp64; positions [axes, T]; cos_sin [max_pos, R]."""
    half = cos_sin.shape[1] // 2
    sections = sections or (half,)
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    pos = positions.clamp(0, cos_sin.shape[0] - 1)
    y = x.double().clone()
    for i in range(half):
        c = cos_sin[pos[axis[i]], i].double()[:, None]
        s = cos_sin[pos[axis[i]], half + i].double()[:, None]
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        xa, xb = x[..., a].double(), x[..., b].double()
        y[..., a], y[..., b] = xa * c - xb * s, xb * c + xa * s
    return y


def attention(q, keys, vals, scale=None, causal=True, window=0):
    """One sequence: q [T, Hq, D], keys and vals [L, Hk, D] (fp64).

    Returns out [T, Hq, D], lse [T, Hq], spread [T, Hq, D] = sum_t p_t |V_t|, and drift [T, Hq] = the
    largest scale * sum_d |q_d K_td| among the tokens seen: what error bounds are made of.
    """
    t, hq, d = q.shape
    n, hk = keys.shape[0], keys.shape[1]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    pos = n - t + torch.arange(t, device=q.device)
    at = torch.arange(n, device=q.device)
    seen = torch.ones(t, n, dtype=torch.bool, device=q.device)
    if causal:
        seen &= at[None] <= pos[:, None]
    if window:
        seen &= at[None] > pos[:, None] - window
    k = keys.repeat_interleave(hq // hk, 1).permute(1, 0, 2)      # [Hq, L, D]
    v = vals.repeat_interleave(hq // hk, 1).permute(1, 0, 2)
    x = q.double().permute(1, 0, 2)                               # [Hq, T, D]
    s = (x @ k.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1) if n else torch.full((hq, t), -math.inf, dtype=torch.float64, device=q.device)
    p = torch.where(seen, torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[..., None]), 0.0)
    drift = (x.abs() @ k.abs().transpose(1, 2) * abs(scale)).masked_fill(~seen, 0.0)
    drift = drift.amax(-1) if n else torch.zeros_like(lse)
    return ((p @ v).permute(1, 0, 2), lse.T, (p @ v.abs()).permute(1, 0, 2), drift.T)

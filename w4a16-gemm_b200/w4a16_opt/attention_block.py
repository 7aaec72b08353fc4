"""An attention block served from 4-bit weights and a 4-bit cache, and a command that runs it.

    PYTHONPATH=w4a16-gemm_b200 python -m w4a16_opt.attention_block [--batch B] [--prompt N] [--steps K]

The block is what stands between two residual additions of a decoder: QKV projection
(``w4a16_gemm``), rotary positions and the quantised write of keys and values (``cache_append``),
attention over the cache (``cache_attention``), output projection.  The command fills a batch of
prompts of different lengths in one call and then decodes token by token from a captured CUDA
graph, with random weights of the Llama-3-8B attention shapes.
"""
from __future__ import annotations

import argparse

import torch

from . import quantize_pack, w4a16_gemm
from .kvcache import Int4KVCache, cache_append, cache_attention


def rotary_table(max_pos: int, rotary_dim: int, theta: float = 500000.0, device=None) -> torch.Tensor:
    """fp32 [max_pos, rotary_dim]: cosines, then sines, of position * theta^(-2i / rotary_dim)."""
    half = rotary_dim // 2
    rate = theta ** (-torch.arange(half, dtype=torch.float64) / half)
    angle = torch.arange(max_pos, dtype=torch.float64)[:, None] * rate
    return torch.cat((angle.cos(), angle.sin()), -1).float().to(device or "cuda")


def slots_of(page_table: torch.Tensor, sequence: torch.Tensor, positions: torch.Tensor, page_size: int) -> torch.Tensor:
    """Cache slots (int64) of tokens, by their sequence and position (int64 tensors of one shape).

    A position that the table has no column for gets slot -1, which an append skips.
    """
    width = page_table.shape[1]
    if width == 0:
        return torch.full_like(positions, -1)
    column = positions // page_size
    inside = column.clamp(0, width - 1)
    slot = torch.add(positions % page_size, page_table[sequence, inside], alpha=page_size)
    return slot.masked_fill_(column != inside, -1)


class AttentionBlock:
    """Projections ``wqkv`` and ``wo`` as (packed words, scales), a cache, and a rotary table."""

    def __init__(self, wqkv, wo, q_heads: int, cache: Int4KVCache, cos_sin: torch.Tensor):
        self.wqkv, self.wo, self.q_heads, self.cache, self.cos_sin = wqkv, wo, q_heads, cache, cos_sin

    def __call__(self, x, positions, slots, page_table, seq_lens, cu_q=None, max_q=None, **mask):
        """x fp16 [tokens, hidden] -> fp16 [tokens, hidden]; see cache_append and cache_attention."""
        hq, hk, d = self.q_heads, self.cache.kv_heads, self.cache.head_dim
        qkv = w4a16_gemm(self.wqkv[0], x, self.wqkv[1]).view(x.shape[0], hq + 2 * hk, d)
        q = cache_append(self.cache, qkv[:, hq:hq + hk], qkv[:, hq + hk:], slots, q=qkv[:, :hq], positions=positions,
                         cos_sin=self.cos_sin)
        y = cache_attention(q, self.cache, page_table, seq_lens, cu_q=cu_q, max_q=max_q, **mask)
        return w4a16_gemm(self.wo[0], y.view(x.shape[0], hq * d), self.wo[1])


class DecodeLoop:
    """One-token steps of a batch from a captured graph: lengths, positions and slots live on the device.

    The loop keeps the caller's ``page_table`` and ``seq_lens`` and counts the latter up in place, one a step;
    the caller may change both between steps (a finished sequence's place given to another).  A step for
    which some sequence's table has no column is refused.
    """

    def __init__(self, block: AttentionBlock, x: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor):
        self.block, self.x, self.page_table, self.seq_lens = block, x.clone(), page_table, seq_lens
        self._left = self._room()
        self._sequence = torch.arange(x.shape[0], device=x.device)
        self._step()                                        # set-up calls happen outside the capture
        self.seq_lens -= 1
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.out = self._step()

    def _room(self) -> int:
        """Steps until the longest sequence fills its table, at least one (waits for the device)."""
        most = self.page_table.shape[1] * self.block.cache.page_size
        room = most - int(self.seq_lens.max()) if self.seq_lens.numel() else most
        if room <= 0:
            raise RuntimeError(f"no step is left: a sequence fills its page table ({most} tokens)")
        return room

    def _step(self):
        positions = self.seq_lens.long()
        slots = slots_of(self.page_table, self._sequence, positions, self.block.cache.page_size)
        self.seq_lens += 1
        return self.block(self.x, positions, slots, self.page_table, self.seq_lens)

    def step(self, x: torch.Tensor) -> torch.Tensor:
        """Appends one token a sequence and returns the block's output (valid until the next step)."""
        if self._left == 0:                                 # or fewer sequences than there were: look again
            self._left = self._room()
        self._left -= 1
        self.x.copy_(x)
        self.graph.replay()
        return self.out


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=2000, help="longest prompt; the others are shorter")
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--page-size", type=int, default=64)
    ap.add_argument("--group-size", type=int, default=128)
    args = ap.parse_args(argv)
    hidden, hq, hk, d, b = 4096, 32, 8, 128, args.batch
    gen = torch.Generator(device="cuda").manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")     # noqa: E731
    wqkv = quantize_pack(rand((hq + 2 * hk) * d, hidden) * 0.02, 128)
    wo = quantize_pack(rand(hidden, hq * d) * 0.02, 128)
    lens = [max(1, args.prompt - args.prompt * i // (2 * b)) for i in range(b)]
    pages = -(-(args.prompt + args.steps + 1) // args.page_size)
    cache = Int4KVCache(b * pages, hk, d, args.page_size, args.group_size)
    block = AttentionBlock(wqkv, wo, hq, cache, rotary_table(args.prompt + args.steps + 1, d))
    table = torch.randperm(b * pages, generator=gen, device="cuda").to(torch.int32).view(b, pages)
    seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    cu_q = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
    sequence = torch.repeat_interleave(torch.arange(b, device="cuda"), seq_lens.long())
    positions = torch.cat([torch.arange(n, device="cuda") for n in lens])
    slots = slots_of(table, sequence, positions, args.page_size)
    x = rand(sum(lens), hidden).half()

    def timed(f):
        f()
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        y = f()
        end.record()
        end.synchronize()
        return y, start.elapsed_time(end) * 1e3

    y, us = timed(lambda: block(x, positions, slots, table, seq_lens, cu_q=cu_q, max_q=max(lens)))
    print(f"prompts: {b} sequences, {sum(lens)} tokens: {us:.0f} us")
    loop = DecodeLoop(block, y[:b], table, seq_lens)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    y = loop.step(y[:b])
    start.record()
    for _ in range(args.steps - 1):
        y = loop.step(y)
    end.record()
    end.synchronize()
    us = start.elapsed_time(end) * 1e3 / max(1, args.steps - 1)
    bits = 8 * cache.data.shape[2] / (2 * args.page_size * d)
    print(f"decode: {args.steps} steps, {us:.1f} us a step; cache {bits:.2f} bits a value, finite: {bool(y.isfinite().all())}")


if __name__ == "__main__":
    main()

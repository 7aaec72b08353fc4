"""A paged key/value cache held in 4 bits: writing it, reading it back, attention over it.

    cache = Int4KVCache(num_pages, kv_heads, head_dim)
    q = cache_append(cache, k, v, slots, q=q, positions=positions, cos_sin=cos_sin)
    y = cache_attention(q, cache, page_table, seq_lens)                      # one token a sequence
    y = cache_attention(q, cache, page_table, seq_lens, cu_q=cu_q, max_q=n)  # prompts, drafts

These are what a decoder served with ``w4a16_gemm`` needs between its QKV and its output
projection; the reference has no counterpart.  Activations are fp16 or bf16 ``[tokens, heads,
head_dim]`` with a dense last dimension (views of a fused QKV output will do).  Every function
runs on the current CUDA stream, and raises RuntimeError on bad input.
"""
from __future__ import annotations

import math

import torch

from . import _C


class Int4KVCache:
    """A paged 4-bit cache: one uint8 tensor ``data`` [num_pages, kv_heads, page_bytes].

    A block (one page, one head) holds the codes of the keys [page_size, head_dim / 2], those
    of the values, and the fp16 pairs (scale, minimum) of the keys [page_size, head_dim /
    group_size, 2] and of the values; byte i of a token's codes is value 2i in its low and value
    2i + 1 in its high four bits, and a value is code * scale + minimum.  Slot ``s`` is row
    ``s % page_size`` of page ``s // page_size``.

    head_dim is 64 or 128, group_size 64 or 128 and at most head_dim (default: head_dim),
    page_size 16, 32, 64, 128 or 256.
    """

    __slots__ = ("data", "head_dim", "page_size", "group_size")

    def __init__(self, num_pages: int, kv_heads: int, head_dim: int, page_size: int = 64,
                 group_size: int | None = None, device=None):
        group_size = head_dim if group_size is None else group_size
        nbytes = _C.cache_page_bytes(page_size, head_dim, group_size)
        self.data = torch.zeros(num_pages, kv_heads, nbytes, dtype=torch.uint8, device=device or "cuda")
        self.head_dim, self.page_size, self.group_size = head_dim, page_size, group_size

    @classmethod
    def wrap(cls, data: torch.Tensor, head_dim: int, page_size: int = 64,
             group_size: int | None = None) -> "Int4KVCache":
        """A cache over memory that the caller keeps (uint8 [num_pages, kv_heads, page_bytes])."""
        self = cls.__new__(cls)
        group_size = head_dim if group_size is None else group_size
        nbytes = _C.cache_page_bytes(page_size, head_dim, group_size)
        if data.dtype != torch.uint8 or data.dim() != 3 or data.shape[2] != nbytes or not data.is_contiguous():
            raise RuntimeError(f"the cache must be a contiguous uint8 [pages, kv_heads, {nbytes}] tensor")
        self.data = data
        self.head_dim, self.page_size, self.group_size = head_dim, page_size, group_size
        return self

    @property
    def num_pages(self) -> int:
        return self.data.shape[0]

    @property
    def kv_heads(self) -> int:
        return self.data.shape[1]


def cache_append(cache: Int4KVCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, *,
                 q: torch.Tensor | None = None, positions: torch.Tensor | None = None,
                 cos_sin: torch.Tensor | None = None, sections=None, interleaved: bool = False):
    """Quantises ``k`` and ``v`` [tokens, kv_heads, head_dim] into ``slots`` (int64 [tokens]).

    A slot outside the cache (-1, say) is skipped; what equal slots of one call leave is
    unspecified (codes of one token may meet scales of another).  Values are clamped to +-57344 and NaN becomes
    0, so that whatever is read back is finite.

    ``positions`` (int64 [tokens], or [axes, tokens] with up to three axes) and ``cos_sin`` (fp32
    [max_pos, rotary_dim]: cosines, then sines; rotary_dim is head_dim or half of it) turn the
    keys before they are quantised, and ``q`` [tokens, q_heads, head_dim], which is returned
    turned.  The pair of angle i is values (i, i + rotary_dim / 2), or (2i, 2i + 1) if
    ``interleaved``.  With several axes, ``sections`` says how many angles each of them has, in
    order.  Positions are clamped into the table.
    """
    return _C.cache_append(cache.data, cache.head_dim, cache.page_size, cache.group_size, k, v, slots, q, positions,
                           cos_sin, sections, interleaved)


def cache_read(cache: Int4KVCache, slots: torch.Tensor, dtype: torch.dtype = torch.float16):
    """Keys and values of ``slots`` (int64 [tokens]) as fresh [tokens, kv_heads, head_dim] tensors.

    ``dtype`` is fp16 or bf16; a slot outside the cache gives zeros.
    """
    if dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError("dtype must be fp16 or bf16")
    return _C.cache_read(cache.data, cache.head_dim, cache.page_size, cache.group_size, slots,
                         dtype == torch.bfloat16)


def cache_attention(q: torch.Tensor, cache: Int4KVCache, page_table: torch.Tensor, seq_lens: torch.Tensor, *,
                    cu_q: torch.Tensor | None = None, max_q: int | None = None, scale: float | None = None,
                    causal: bool = True, window: int = 0, return_lse: bool = False,
                    out: torch.Tensor | None = None, workspace: torch.Tensor | None = None):
    """softmax(scale * q K^T + mask) V over each sequence's cached tokens; fresh, or into ``out``.

    ``q`` [tokens, q_heads, head_dim], q_heads a multiple of the cache's kv_heads.  ``page_table``
    int32 [batch, pages] lists each sequence's pages in order (entries past its end are not used),
    ``seq_lens`` int32 [batch] its cached tokens, those of the queries included.  ``cu_q`` int32
    [batch + 1] says where each sequence's queries start in ``q`` and ``max_q`` how many the
    longest has (any number above it will do too); without ``cu_q`` there is one for each.  Rows
    that belong to no sequence, as in a captured step of fixed size, and queries of a sequence past
    its first ``max_q`` give zeros (and -inf, below).

    Query i of the T of a sequence of L tokens has position L - T + i.  It sees every token of
    the sequence, with ``causal`` those up to its position, with ``window`` > 0 those above its
    position - window.  A query that sees none gives zeros, and -inf in the log of the sum of
    exponentials (fp32 [tokens, q_heads]) that comes second with ``return_lse``.

    The lengths stay on the device, and the call is planned by the sizes of its arguments.  A table of
    far more columns than the sequences use makes prompts slower: a view of the columns in use will
    do.  More than 32 rows (``max_q`` times the query heads that share a key head) send the whole
    call to the kernel for prompts, where single tokens are slow: give them a call of their own.

    ``scale`` defaults to 1 / sqrt(head_dim).  ``workspace``: optional scratch CUDA buffer
    (256-byte aligned); without it the binding keeps one per (device, stream).
    """
    if max_q is None:
        if cu_q is not None:
            raise RuntimeError("cu_q needs max_q, the largest number of queries of a sequence")
        max_q = 1
    max_q = min(max_q, q.shape[0])
    y, lse = _C.cache_attention(q, cache.data, cache.head_dim, cache.page_size, cache.group_size, page_table, seq_lens,
                                cu_q, max_q, 1.0 / math.sqrt(cache.head_dim) if scale is None else scale, causal,
                                window, return_lse, out, workspace)
    return (y, lse) if return_lse else y

"""Generation: a paged cache of keys and values in 8 bits, and attention over it.

A cache is a pool of pages; a page holds ``page_size`` tokens of every kv head, one byte a value, with one scale for
each head's keys and one for its values.  Which page holds which tokens of a sequence is the caller's ``page_table``:
position ``p`` of sequence ``b`` is slot ``p % page_size`` of page ``page_table[b, p // page_size]``.  Entries outside of
the pool (``-1``) hold no tokens: nothing is written there, and no row sees them.

The reference has no counterpart: its operator takes dense 16-bit keys and values.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from .interface import _native_host

__all__ = ["QuantizedKVCache", "kv_cache_write", "kv_cache_read", "kv_cache_attention"]


@dataclass
class QuantizedKVCache:
    """``k`` [num_pages, Hkv, page_size, d] and ``v`` [num_pages, Hkv, page_size, dv], both ``float8_e4m3fn`` or both ``int8``;
    ``k_scale`` and ``v_scale`` [num_pages, Hkv] fp32; contiguous.  A stored value is payload x scale.

    Scales are powers of two, the least that bring the largest magnitude of the page's tokens into the payload's range
    (448 or 127): reading back is exact, and the only error is the payload's rounding, half of 2^-3 of the value in e4m3,
    half a scale in int8.  Served: page sizes 16, 32, 64 and 128; head dims up to 128 in steps of 16, 192 / 128, 256 / 256."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def empty(cls, num_pages: int, num_kv_heads: int, head_dim: int, head_dim_v: Optional[int] = None, *, page_size: int = 64,
              dtype: torch.dtype = torch.float8_e4m3fn, device="cuda") -> "QuantizedKVCache":
        """A cache of zeros."""
        if dtype not in (torch.float8_e4m3fn, torch.int8):
            raise TypeError(f"the cache holds float8_e4m3fn or int8, got {dtype}")
        if page_size not in (16, 32, 64, 128):
            raise NotImplementedError(f"page_size {page_size} is not 16, 32, 64 or 128")
        dv = head_dim if head_dim_v is None else head_dim_v
        if head_dim % 16 or dv % 16 or not ((0 < head_dim <= 128 and 0 < dv <= 128) or (head_dim, dv) in ((192, 128), (256, 256))):
            raise NotImplementedError(f"head dims {head_dim} / {dv}: multiples of 16 up to 128, 192 / 128 and 256 / 256 are served")
        k = torch.zeros(num_pages, num_kv_heads, page_size, head_dim, dtype=torch.uint8, device=device).view(dtype)
        v = torch.zeros(num_pages, num_kv_heads, page_size, dv, dtype=torch.uint8, device=device).view(dtype)
        scales = [torch.full((num_pages, num_kv_heads), 2.0 ** -64, dtype=torch.float32, device=device) for _ in range(2)]
        return cls(k, v, *scales)

    @property
    def page_size(self) -> int:
        return self.k.shape[2]


def kv_cache_write(cache: QuantizedKVCache, key: torch.Tensor, value: torch.Tensor, page_table: torch.Tensor, start: torch.Tensor,
                   lengths: Optional[torch.Tensor] = None) -> None:
    """Rounds ``key`` [B, S, Hkv, d] and ``value`` [B, S, Hkv, dv] (bf16 / fp16) into the cache: row i of sequence b goes to
    position ``start[b] + i``, for ``i < lengths[b]`` (all rows without ``lengths``).  ``page_table`` [B, n], ``start`` and
    ``lengths`` [B] are int32.

    A page whose first slot is written begins anew.  Where a write begins inside a page, the page's scale stays or
    grows with the new tokens; when it grows, the earlier tokens are rounded again on the new grid (in e4m3 that moves
    only values that become subnormal).  Slots behind the last token are left as they are.  A NaN or an infinity reads back
    as NaN; in int8 so does the whole page of that head, until the page begins anew.  Magnitudes below about 2^-73 (e4m3) or
    2^-65 (int8) become zero, those near the end of bf16's range saturate.  A page must not be written for two sequences in
    one call, nor appear twice in the row that one writes through; pages that sequences share are written once and then only read."""
    _native_host().kv_write(cache.k, cache.v, cache.k_scale, cache.v_scale, key, value, page_table, start, lengths)


def kv_cache_read(cache: QuantizedKVCache, page_table: torch.Tensor, start: torch.Tensor, seqlens: torch.Tensor, length: int, *,
                  dtype: torch.dtype = torch.bfloat16):
    """(key [B, length, Hkv, d], value [B, length, Hkv, dv]): the tokens at positions ``start[b] + i``; zeros where that is
    negative or not below ``seqlens[b]``.  Exact in bf16; in fp16 magnitudes beyond 65504 saturate, and below 2^-14 they are rounded to multiples of 2^-24."""
    if dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"kv_cache_read gives bfloat16 / float16, got {dtype}")
    return _native_host().kv_read(cache.k, cache.v, cache.k_scale, cache.v_scale, page_table, start, seqlens, length,
                                  dtype == torch.float16)


def kv_cache_attention(query: torch.Tensor, cache: QuantizedKVCache, page_table: torch.Tensor, seqlens: torch.Tensor, *,
                       q_lengths: Optional[torch.Tensor] = None, causal: bool = True, window_size: Optional[int] = None,
                       softmax_scale: Optional[float] = None, sink: Optional[torch.Tensor] = None,
                       learnable_sink: Optional[torch.Tensor] = None, max_seqlen: Optional[int] = None, return_lse: bool = False,
                       return_softmax_lse: bool = False):
    """Attention of ``query`` [B, S, Hq, d] (bf16 / fp16) over the cached tokens, without gradients: ``out`` [B, S, Hq, dv],
    or ``(out, lse)`` with ``lse`` [B, Hq, S] fp32.

    ``seqlens`` [B] int32 counts every sequence's tokens, the queries' own included (write them first).  Sequence b has
    ``n = q_lengths[b]`` query rows (S without ``q_lengths``; the rest is padding), and row i stands at position
    ``seqlens[b] - n + i``.  It sees the positions up to its own, with ``window_size`` the last ``window_size`` of them, or all
    without ``causal``.  Rows that see nothing, padding among them, give 0 and an lse of -inf (of the sink's logit with
    ``sink``, one per query head, which joins every denominator).  A NaN reaches the rows that see its token and no others: a
    NaN value in e4m3 its column, a NaN key, and in int8 a page whose scale is NaN, the whole row and its lse.

    Up to 96 rows for each kv head (S x Hq / Hkv; more with head dims above 128 and few kv heads in all sequences together) the pages
    are read as they are, and neither ``seqlens`` nor anything else is needed on the host, so the call can be captured into a CUDA graph
    with lengths that change between replays.  With more rows the tokens are read back into 16-bit tensors of ``max_seqlen`` positions
    (an upper bound of ``seqlens``; without it the
    whole page table, as long as that takes no more than 2 GiB: the call's time goes with these positions, tokens or not), with a window no more than its last S + ``window_size`` - 1, and go through the dense forward; more positions than it takes (262144 at
    head dims other than 256) stay with the pages.  At most 1024 sequences where the pages are read as they are.

    Precision: sums and statistics are fp32.  Where the pages are read as they are, the weights p are rounded to fp16 (half a step is 2^-11) whatever query's
    type, and keys and values are exact; the dense forward rounds p to query's type (2^-8 in bf16) and takes the tokens as ``kv_cache_read`` gives them in
    that type, so with fp16 queries values of a cache that was written in bf16 saturate and lose small magnitudes as they do there."""
    if sink is not None and learnable_sink is not None:
        raise ValueError("pass either sink or learnable_sink, not both")
    if window_size is not None and window_size < 1:
        raise ValueError("window_size needs causal=True and at least one token")
    if max_seqlen is not None and max_seqlen < 0:
        raise ValueError("max_seqlen must not be negative")
    out, lse = _native_host().kv_attention(query, cache.k, cache.v, cache.k_scale, cache.v_scale, page_table, seqlens, q_lengths,
                                           sink if sink is not None else learnable_sink, bool(causal), window_size or 0, softmax_scale,
                                           1 << 40 if max_seqlen is None else max_seqlen)
    return (out, lse) if return_lse or return_softmax_lse else out

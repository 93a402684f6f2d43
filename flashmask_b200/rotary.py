"""What stands before attention: RMS norm of every head of q and k, and their rotation by position, in one pass.

The reference has no counterpart: it begins at attention.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .interface import _native_host

__all__ = ["qk_norm_rotary"]


def qk_norm_rotary(query: torch.Tensor, key: torch.Tensor, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
                   cos: torch.Tensor, sin: torch.Tensor, positions: Optional[torch.Tensor] = None, *, eps: float = 1e-6,
                   interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """``query`` [B, S, Hq, d] and ``key`` [B, S, Hk, d] (bf16 / fp16, any strides: views of a fused projection are read in
    place) -> new tensors of the same shapes, ready for ``flashmask_attention`` or ``kv_cache_write``.

    Every row x of d values becomes ``u = x / sqrt(mean(x^2) + eps) * weight`` with ``q_weight`` / ``k_weight`` [d] (fp32 or
    query's dtype; None: ones).  Then the pairs (a, b) of its first ``2 n`` values turn into ``(a cos - b sin, b cos + a sin)``
    with the rows of ``cos`` and ``sin`` (fp32 [positions, n], n a multiple of 8) at the token's position; pairs are
    ``(i, i + n)``, or ``(2 i, 2 i + 1)`` with ``interleaved``.  ``positions`` (int32 / int64, [B, S] or [S]) says where tokens
    stand, e.g. from 0 in every packed document; without it token i stands at i.  A position that the tables do not have makes its rows
    NaN, what does not turn included (with n = 0 positions say nothing).  Sums and products are fp32, rounded once.

    Gradients of query, key and the weights are exact to the same rounding and bitwise reproducible; they have no gradients themselves.
    There is no forward-mode derivative: dual tensors are refused."""
    return _native_host().norm_rotary(query, key, q_weight, k_weight, cos, sin, positions, eps, interleaved)

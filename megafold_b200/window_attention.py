"""Attention with a sliding window and a few first tokens that stay visible (sinks).

Stands beside ``TritonEvoformer`` for sequences whose pair bias would be too large: long chains, chunks of a long row
behind the keys before them, single queries.  It is not the reference's attention over atoms (megafold/model/attention.py:260-394, in torch
there), which adds a pair bias and gives one window to a whole block of queries: here each query has a window of its own, and there is no bias.
The work is done by the CUDA library (``mf_window_fwd`` / ``mf_window_bwd``); tensors on any other device are rejected.
"""
from __future__ import annotations

from . import _lib

__all__ = ["window_attention", "window_attention_forward", "window_attention_backward"]

_NO_BOUND = 2 ** 31 - 1


def _span(left, right, sinks):
    return _NO_BOUND if left is None else left, _NO_BOUND if right is None else right, sinks


def window_attention(Q, K, V, left, right=0, sinks: int = 0, mask=None):
    """Q: ``[B, N, Lq, H, D]``; K, V: ``[B, N, Lk, Hk, D]``, H a multiple of Hk (query head h reads key head ``h // (H // Hk)``); D at most 128.

    Query i stands at position ``p = i + Lk - Lq`` (the queries are the last of the keys) and sees key j where ``j <= p + right`` and
    ``j >= p - left`` or ``j < sinks``.  ``left`` or ``right`` None: no bound on that side; ``right=0`` is causal.
    mask: a bool (or uint8) keep-mask ``[B, N, 1, 1, Lk]``.  What keys hold that are masked or that no query sees, even NaN, reaches
    nothing.  A query that sees no key gives zeros and passes no gradient.

    float32 tensors, and 16-bit ones whose head size is no multiple of 8 or whose rows are not 16-byte aligned, run on the CUDA cores: right at every
    size, and far ahead of a masked product where windows are narrow, but no faster than library products where a window is about as wide as the
    sequence."""
    return _lib.native().window_attention(Q, K, V, mask, *_span(left, right, sinks))


def window_attention_forward(q, k, v, left, right=0, sinks: int = 0, mask=None, flags: int = 0):
    """Returns ``(O [B, N, Lq, H, D], LSE fp32 [B, N, H, Lq])``; ``mf_window_fwd`` of the C ABI."""
    return _lib.native().window_forward(q, k, v, mask, *_span(left, right, sinks), flags)


def window_attention_backward(d_o, q, k, v, o, lse, left, right=0, sinks: int = 0, mask=None, flags: int = 0):
    """Returns ``(dQ, dK, dV)``; ``mf_window_bwd``.  Every sum has a fixed order: the results are bit-reproducible."""
    return _lib.native().window_backward(d_o, q, k, v, mask, *_span(left, right, sinks), o, lse, flags)

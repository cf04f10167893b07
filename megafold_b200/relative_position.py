"""Learned relative position bias by buckets: the pair bias of an attention from a table, with the table's gradient.

``relative_position_bias`` gives the ``[B, 1, H, Lq, Lk]`` tensor that ``TritonEvoformer`` takes as ``pair_bias``; its gradient comes
back as the table's.  Two ways to put distances into buckets:

* ``"clip"``: a bucket for each distance from ``-max_distance`` to ``max_distance``, farther ones in the outermost.  The relative position
  encoding of the pair representation (megafold/model/megafold.py, ``RelativePositionEncoding``) has the same buckets in the other order: it
  clips query minus key, this key minus query.  A table that was learned there arrives mirrored: ``table[:2 * max_distance + 1].flip(0)``
  brings its buckets into this order (a last row for other chains stays where it is);
* ``"log"``: one bucket for each small distance, then buckets that grow by a constant ratio up to ``max_distance``; with
  ``bidirectional`` half of them for keys behind the query, half for keys before it.

The borders of logarithmic buckets are computed in whole numbers, so that a distance on a border has one answer.
The work is done by the CUDA library (``mf_relpos_fwd`` / ``mf_relpos_bwd``); tensors on any other device are rejected.
"""
from __future__ import annotations

import functools

import torch
from torch import nn

from . import _lib

__all__ = ["relative_position_bias", "RelativePositionBias"]

MAX_DISTANCE = 16384
MAX_ROWS = 1024


@functools.lru_cache(maxsize=256)
def _buckets(count: int, max_distance: int, scheme: str, bidirectional: bool):
    """``(edges, (base_pos, step_pos, base_neg, step_neg))``: with ``m`` edges at or below ``|d|`` the bucket of the distance ``d`` is
    ``base_pos + step_pos * m`` for ``d > 0``, else ``base_neg + step_neg * m``."""
    if max_distance < 1 or max_distance > MAX_DISTANCE:
        raise ValueError(f"max_distance must be between 1 and {MAX_DISTANCE}, got {max_distance}")
    if scheme == "clip":
        if count != (2 * max_distance + 1 if bidirectional else max_distance + 1):
            raise ValueError(f"distances clipped to {max_distance} take {2 * max_distance + 1} buckets, {max_distance + 1} in one direction, got {count}")
        return tuple(range(1, max_distance + 1)), ((max_distance, 1, max_distance, -1) if bidirectional else (0, 0, 0, 1))
    if scheme != "log":
        raise ValueError(f"scheme must be 'log' or 'clip', got {scheme!r}")
    if bidirectional and count % 2:
        raise ValueError(f"two directions take an even number of buckets, got {count}")
    side = count // 2 if bidirectional else count
    near = side // 2
    if near < 1 or max_distance <= near:
        raise ValueError(f"{count} buckets and max_distance {max_distance} leave no logarithmic bucket")
    edges = list(range(1, near + 1))
    steps = side - near
    for k in range(1, steps):
        # the smallest n with near + floor(log(n / near) / log(max_distance / near) * steps) >= near + k
        lo, hi = near, max_distance
        while lo < hi:
            n = (lo + hi) // 2
            if n ** steps * near ** k >= max_distance ** k * near ** steps:
                hi = n
            else:
                lo = n + 1
        edges.append(lo)
    return tuple(edges), ((side, 1, 0, 1) if bidirectional else (0, 0, 0, 1))


def _check_rows(rows: int):
    if rows > MAX_ROWS:
        raise ValueError(f"a table of at most {MAX_ROWS} rows is supported, got {rows}")


def relative_position_bias(weight, q_positions, k_positions, *, max_distance: int, scheme: str = "log", bidirectional: bool = True, q_segments=None,
                           k_segments=None, dtype=None):
    """``[B, 1, H, Lq, Lk]``: ``weight[bucket(k_positions[b, j] - q_positions[b, i]), h]``.

    weight: ``[buckets, H]``, with segments ``[buckets + 1, H]``, whose last row is that of pairs from different segments (chains).
    q_positions, k_positions: int32 or int64, ``[Lq]`` / ``[Lk]`` or ``[B, Lq]`` / ``[B, Lk]``; or two numbers, the lengths of rows whose
    queries are the last of the keys; differences of positions have to fit 64 bits.  dtype: of the result, ``weight.dtype`` by default.  One direction
    (``bidirectional=False``): keys ahead of the query share the bucket of distance 0."""
    if weight.dim() != 2:
        raise ValueError(f"weight must be [rows, heads], got {tuple(weight.shape)}")
    _check_rows(weight.shape[0])
    if isinstance(q_positions, int) != isinstance(k_positions, int):
        raise TypeError("positions are two tensors or two lengths")
    edges, rows = _buckets(weight.shape[0] - (q_segments is not None), int(max_distance), scheme, bool(bidirectional))
    if isinstance(q_positions, int):
        return _lib.native().relative_position_bias(weight, None, None, q_positions, k_positions, q_segments, k_segments, edges, rows, dtype)
    return _lib.native().relative_position_bias(weight, q_positions, k_positions, 0, 0, q_segments, k_segments, edges, rows, dtype)


class RelativePositionBias(nn.Module):
    """The table ``weight`` as a parameter, ``num_buckets`` rows (with ``segments`` one more) of ``num_heads`` values."""

    def __init__(self, num_heads, num_buckets=32, max_distance=128, scheme="log", bidirectional=True, segments=False, device=None, dtype=None):
        super().__init__()
        _check_rows(num_buckets + bool(segments))
        _buckets(num_buckets, max_distance, scheme, bool(bidirectional))
        self.max_distance, self.scheme, self.bidirectional, self.segments = max_distance, scheme, bool(bidirectional), segments
        self.weight = nn.Parameter(torch.empty(num_buckets + bool(segments), num_heads, device=device, dtype=dtype))
        nn.init.normal_(self.weight, std=0.02)

    def forward(self, q_positions, k_positions, q_segments=None, k_segments=None, dtype=None):
        if self.segments != (q_segments is not None):
            raise ValueError("the table has a row for pairs of different segments" if self.segments else "the table has no row for pairs of different segments")
        return relative_position_bias(self.weight, q_positions, k_positions, max_distance=self.max_distance, scheme=self.scheme,
                                      bidirectional=self.bidirectional, q_segments=q_segments, k_segments=k_segments, dtype=dtype)

    def extra_repr(self):
        return f"rows={self.weight.shape[0]}, num_heads={self.weight.shape[1]}, max_distance={self.max_distance}, scheme={self.scheme!r}"

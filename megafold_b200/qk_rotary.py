"""RMS norm of every head of queries and keys and their rotation by position, in one pass over both.

For attention on ``[B, N, L, H, D]`` tensors: what comes out goes to ``TritonEvoformer`` or ``window_attention``, what goes in may be
strided views of a merged projection.  Angles are formed in 64 bits, so positions of millions keep their fractions of a
turn.  The work is done by the CUDA library (``mf_qk_rotary_fwd`` / ``mf_qk_rotary_bwd``); tensors on any other device are rejected.
"""
from __future__ import annotations

import torch
from torch import nn

from . import _lib

__all__ = ["qk_norm_rotary", "QKNormRotary"]


def qk_norm_rotary(q, k, q_weight, k_weight, inv_freq, positions=None, eps: float = 1e-6, interleaved: bool = False):
    """Returns ``(q', k')``, contiguous: each head ``x * (mean(x^2) + eps)^-1/2 * weight``, then the pairs of its first ``2 * len(inv_freq)``
    elements turned by ``position * inv_freq``.

    q: ``[B, N, L, H, D]``, k: ``[B, N, L, Hk, D]``; D at most 256.  q_weight, k_weight: ``[D]``, or ``[H, D]`` and ``[Hk, D]`` for a weight
    of each head, or None both.  inv_freq: float32 ``[R / 2]``, no gradient.  positions: int32 or int64 ``[L]``, ``[N, L]`` or ``[B, N, L]``;
    None: 0, 1, ... along L.  eps: taken in 32 bits; 0 is fine for heads that are not all zeros.  interleaved: pairs are neighbours
    (2i, 2i + 1) instead of (i, i + R / 2)."""
    return _lib.native().qk_norm_rotary(q, k, q_weight, k_weight, inv_freq, positions, eps, interleaved)


class QKNormRotary(nn.Module):
    """The weights ``q_weight`` and ``k_weight`` as parameters, shared by the heads or (with ``num_heads``) one for each head."""

    def __init__(self, head_dim, rotary_dim=None, num_heads=None, num_key_heads=None, base=10000.0, interleaved=False, eps=1e-6, device=None, dtype=None):
        super().__init__()
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if rotary_dim % 2 or not 0 <= rotary_dim <= head_dim:
            raise ValueError(f"{rotary_dim} of {head_dim} elements cannot be rotated in pairs")
        self.rotary_dim, self.base, self.interleaved, self.eps = rotary_dim, base, interleaved, eps
        num_key_heads = num_heads if num_key_heads is None else num_key_heads
        self.q_weight = nn.Parameter(torch.empty(*(() if num_heads is None else (num_heads,)), head_dim, device=device, dtype=dtype))
        self.k_weight = nn.Parameter(torch.empty(*(() if num_heads is None else (num_key_heads,)), head_dim, device=device, dtype=dtype))
        self.register_buffer("inv_freq", self._frequencies(device), persistent=False)
        self.reset_parameters()

    def reset_parameters(self) -> None:
        nn.init.ones_(self.q_weight)
        nn.init.ones_(self.k_weight)

    def _frequencies(self, device):
        # on the host, whatever device is the default at the time of a call with one
        steps = torch.arange(0, self.rotary_dim, 2, dtype=torch.float64, device=None if device is None else "cpu")
        freq = self.base ** (-steps / max(self.rotary_dim, 1))
        return freq.to(device=device, dtype=torch.float32)

    def _apply(self, fn, recurse=True):
        # Frequencies stay float32 when the module is moved to another type.  They are in no state dict: those of a module built without memory
        # (the meta device) are computed when it gets some, by this call or by weights that load_state_dict assigned.
        if self.inv_freq.is_meta and not self.q_weight.is_meta:
            self.inv_freq = self._frequencies(self.q_weight.device)
        freq = self.inv_freq
        super()._apply(fn, recurse)
        device = self.inv_freq.device
        self.inv_freq = self._frequencies(device) if freq.is_meta and device.type != "meta" else freq.to(device)
        return self

    def forward(self, q, k, positions=None):
        return qk_norm_rotary(q, k, self.q_weight, self.k_weight, self.inv_freq, positions, self.eps, self.interleaved)

    def extra_repr(self):
        return f"head_dim={self.q_weight.shape[-1]}, rotary_dim={2 * self.inv_freq.shape[0]}, interleaved={self.interleaved}"

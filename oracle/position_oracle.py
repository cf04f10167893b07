"""Plain restatements, in 64 bits, of the operators for positions in attention: the oracle of their tests.

``window`` also gives the bounds of the rounding errors of a kernel that keeps sums in 32 bits and rounds probabilities, their
gradients and results to a type of unit roundoff ``u`` (half a step, ``finfo.eps / 2``)."""
import functools
import math

import torch

U32 = 2.0 ** -24


def bucket(d, count, max_distance, scheme, bidirectional):
    """Bucket of one distance, by the definition, in whole numbers."""
    if scheme == "clip":
        return min(max(d, -max_distance), max_distance) + max_distance if bidirectional else min(max(-d, 0), max_distance)
    side = count // 2 if bidirectional else count
    shift = side if bidirectional and d > 0 else 0
    n = abs(d) if bidirectional else max(-d, 0)
    near = side // 2
    if n < near:
        return shift + n
    steps = side - near
    entered = sum(n >= e for e in _entries(near, steps, max_distance))
    return shift + near + entered


@functools.lru_cache(None)
def _entries(near, steps, max_distance):
    """The smallest distances with log(n / near) / log(max_distance / near) * steps >= k, for k = 1 .. steps - 1."""
    out, n = [], near
    for k in range(1, steps):
        while n ** steps < max_distance ** k * near ** (steps - k):
            n += 1
        out.append(n)
    return tuple(out)


@functools.lru_cache(None)
def _table(count, max_distance, scheme, bidirectional):
    return torch.tensor([bucket(x, count, max_distance, scheme, bidirectional) for x in range(-max_distance - 1, max_distance + 2)])


def buckets(q_pos, k_pos, count, max_distance, scheme, bidirectional):
    d = (k_pos[:, None, :] - q_pos[:, :, None]).clamp(-max_distance - 1, max_distance + 1)
    return _table(count, max_distance, scheme, bidirectional)[d + max_distance + 1]


def relpos(weight, rows, d_bias=None):
    """(bias [B, 1, H, Lq, Lk], gradient of the table, sum of the gradient's magnitudes)"""
    w = weight.double()
    bias = w[rows].permute(0, 3, 1, 2).unsqueeze(1)
    if d_bias is None:
        return bias
    d = d_bias.double()[:, 0].permute(0, 2, 3, 1).reshape(-1, w.shape[1])
    grad, size = torch.zeros_like(w), torch.zeros_like(w)
    grad.index_add_(0, rows.reshape(-1), d)
    size.index_add_(0, rows.reshape(-1), d.abs())
    return bias, grad, size


def rotary(x, weight, inv_freq, positions, eps, interleaved):
    """x [B, N, L, H, D], positions broadcastable to [B, N, L]; differentiable"""
    x = x.double()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.double()
    R = 2 * inv_freq.shape[0]
    a = positions.double()[..., None, None] * inv_freq.double()
    c, s = torch.cos(a), torch.sin(a)
    first = torch.arange(R // 2) * 2 if interleaved else torch.arange(R // 2)
    second = first + 1 if interleaved else first + R // 2
    y1, y2 = y[..., first], y[..., second]
    out = y.clone()
    out[..., first] = y1 * c - y2 * s
    out[..., second] = y2 * c + y1 * s
    return out


def seen(Lq, Lk, left, right, sinks):
    p, j = torch.arange(Lq)[:, None] + Lk - Lq, torch.arange(Lk)
    ok = torch.ones(Lq, Lk, dtype=torch.bool)
    if right is not None:
        ok &= j <= p + right
    if left is not None:
        ok &= (j >= p - left) | (j < sinks)
    return ok


def window(q, k, v, left, right, sinks, mask=None, d_o=None, u=U32):
    """A dict of o, lse and, with d_o, dq, dk, dv, each with its bound under the same name + '_tol'."""
    q, k, v = q.double(), k.double(), v.double()
    B, N, Lq, H, D = q.shape
    Lk, Hk = k.shape[2], k.shape[3]
    G = H // Hk
    ok = seen(Lq, Lk, left, right, sinks)[None, None, None].expand(B, N, 1, Lq, Lk)
    if mask is not None:
        keep = mask.bool().expand(B, N, 1, 1, Lk)
        ok = ok & keep
        gone = ~keep.reshape(B, N, Lk, 1, 1)
        k, v = k.masked_fill(gone, 0.0), v.masked_fill(gone, 0.0)
    rows = lambda t: t.permute(0, 1, 3, 2, 4)                                                             # noqa: E731
    Q, K, V = rows(q), rows(k).repeat_interleave(G, 2), rows(v).repeat_interleave(G, 2)
    scale = 1 / math.sqrt(D)
    s = (Q @ K.transpose(-1, -2) * scale).masked_fill(~ok, -math.inf)
    lse = torch.logsumexp(s, -1) if Lk else torch.full(s.shape[:-1], -math.inf, dtype=torch.float64)
    P = torch.exp(s - lse[..., None].masked_fill(lse[..., None] == -math.inf, 0.0))
    o = P @ V
    # 32 bits: a logit is off by at most (D + 4) roundings of the sum of its products' magnitudes, a probability by twice that and
    # the exponential's, sums by a rounding an addend (Lk, a loose bound)
    ds = (D + 4) * U32 * scale * (Q.abs() @ K.abs().transpose(-1, -2)).amax((-1, -2), keepdim=True) if Lk and Lq else torch.zeros(())
    c = 2 * ds + 2.0 ** -20 + Lk * U32
    A = P @ V.abs()
    o_tol = (u + c) * A + u * o.abs() + 1e-30
    back = lambda t: rows(t)                                                                              # noqa: E731
    out = dict(o=back(o), o_tol=back(o_tol), lse=lse, lse_tol=(c * 2).expand(lse.unsqueeze(-1).shape).squeeze(-1) + 4 * U32 * lse.abs().masked_fill(lse == -math.inf, 0.0))
    if d_o is None:
        return out
    dO = rows(d_o.double())
    delta = (dO * o).sum(-1, keepdim=True)
    dP = dO @ V.transpose(-1, -2)
    dS = P * (dP - delta)
    # delta is formed from the rounded o
    d_delta = (dO.abs() * (o_tol + u * o.abs())).sum(-1, keepdim=True)
    size = dO.abs() @ V.abs().transpose(-1, -2) + (dO * o).abs().sum(-1, keepdim=True)
    dS_tol = u * dS.abs() + P * d_delta + (c + (D + Lk) * U32) * P * size
    group = lambda t: t.reshape(B, N, Hk, G, *t.shape[3:]).sum(3)                                         # noqa: E731
    dq = dS @ K * scale
    dk = group(dS.transpose(-1, -2) @ Q) * scale
    dv = group(P.transpose(-1, -2) @ dO)
    more = (Lk + Lq * G) * U32
    dq_tol = scale * ((dS_tol + more * dS.abs()) @ K.abs()) + u * dq.abs()
    dk_tol = scale * group((dS_tol + more * dS.abs()).transpose(-1, -2) @ Q.abs()) + u * dk.abs()
    dv_tol = group(((u + c + more) * P).transpose(-1, -2) @ dO.abs()) + u * dv.abs()
    for name, t, tol in (("dq", dq, dq_tol), ("dk", dk, dk_tol), ("dv", dv, dv_tol)):
        out[name], out[name + "_tol"] = back(t), back(tol) + 1e-30
    return out

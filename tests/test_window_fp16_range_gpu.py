"""Window attention in fp16 with the gradients of a scaled loss: what fits fp16 arrives, although its terms before the factor D^-1/2 do not."""
import math

import pytest
import torch

import test_window_gpu as base
from oracle import position_oracle as orc

HF = torch.float16
CASES = [  # B, N, Lq, Lk, H, D, left, every (a key of so many is kept), graded (queries with a gradient), its size
    (1, 2, 40, 40, 2, 128, 2, 1, 40, 8000),             # a narrow window
    (2, 1, 60, 1500, 2, 128, None, 211, 60, 9000),      # a wide one
    (1, 1, 900, 900, 2, 128, None, 150, 50, 9500),      # sums in parts
]


def _case(B, N, Lq, Lk, H, D, left, every, graded, size):
    q, k, v, _, d_o = base._inputs(B, N, Lq, Lk, H, H, D, "none", HF)
    d_o = (d_o * size).to(HF)
    d_o[:, :, :Lq - graded] = 0
    return q, k, v, torch.arange(Lk).view(1, 1, 1, 1, Lk) % every == 0, d_o


def _largest_ds(q, k, v, mask, d_o, left):
    """The largest of P (dP - delta), of heads that share no keys."""
    Q, K, V, G = (t.double().permute(0, 1, 3, 2, 4) for t in (q, k, v, d_o))
    s = (Q @ K.transpose(-1, -2) / math.sqrt(q.shape[-1])).masked_fill(~(orc.seen(q.shape[2], k.shape[2], left, 0, 0) & mask), -math.inf)
    P = torch.softmax(s, -1)
    dP = G @ V.transpose(-1, -2)
    return float((P * (dP - (P * dP).sum(-1, keepdim=True))).abs().max())


@pytest.mark.parametrize("B,N,Lq,Lk,H,D,left,every,graded,size", CASES)
def test_the_cases_reach_the_range(B, N, Lq, Lk, H, D, left, every, graded, size):
    q, k, v, m, d_o = _case(B, N, Lq, Lk, H, D, left, every, graded, size)
    assert torch.isfinite(d_o).all() and _largest_ds(q, k, v, m, d_o, left) > 65520              # what fp16 rounds to infinity
    ref = orc.window(q, k, v, left, 0, 0, m, d_o, u=2.0 ** -11)
    assert all(float((ref[x].abs() + ref[x + "_tol"]).max()) < 65504 for x in ("dq", "dk", "dv"))


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,Lq,Lk,H,D,left,every,graded,size", CASES)
def test_gradients_of_a_scaled_loss(B, N, Lq, Lk, H, D, left, every, graded, size):
    base._run(*_case(B, N, Lq, Lk, H, D, left, every, graded, size), left, 0, 0)

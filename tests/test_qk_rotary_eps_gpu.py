"""Norm and rotation with eps = 0: rows that hold numbers have finite gradients, whatever the tokens leave of a block's last step."""
import pytest
import torch

import megafold_b200 as mfb
import test_qk_rotary_gpu as base

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32

SIZES = [  # B, N, L, H, Hk, D, R: one token, a few more than a block's step, ragged ones, several chunks
    (1, 1, 1, 4, 4, 32, 32), (1, 1, 9, 4, 4, 32, 32), (2, 3, 17, 4, 4, 32, 16), (1, 1, 5, 32, 8, 128, 128), (3, 5, 61, 5, 1, 24, 10), (2, 20, 131, 4, 4, 32, 32),
    (1, 1, 3001, 16, 4, 64, 64),
]


@pytest.mark.parametrize("eps", [0.0, 1e-50])
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("B,N,L,H,Hk,D,R", SIZES)
def test_no_eps(B, N, L, H, Hk, D, R, dt, per_head, shared, eps):
    """1e-50 is 0 in the 32 bits that the kernel takes it in.  shared: one set of positions for all sequences."""
    q, k, qw, kw, freq, pos, dq, dk = base._inputs(B, N, L, H, Hk, D, R, per_head, dt)
    if shared:
        pos = torch.arange(L).expand(B, N, L)
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, qw, kw)]
    outs = mfb.qk_norm_rotary(*leaves, freq.cuda(), None if shared else pos.cuda(), eps, False)
    grads = torch.autograd.grad(outs, leaves, [dq.cuda(), dk.cuda()])
    assert all(torch.isfinite(t).all() for t in (*outs, *grads))
    base._compare(q, k, qw, kw, freq, pos, dq, dk, 0.0, False, leaves, outs, grads)

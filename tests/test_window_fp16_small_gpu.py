"""Window attention in fp16 with small gradients, and with gradients of very different sizes: dS keeps its eleven bits although the type has five of exponent."""
import pytest
import torch

import megafold_b200 as mfb
import test_window_gpu as base

pytestmark = pytest.mark.gpu
HF = torch.float16


def _exact(q, k, v, d_o, left):
    """dQ, dK, dV in 64 bits, causal."""
    Q, K, V, G = (t.double().permute(0, 1, 3, 2, 4) for t in (q, k, v, d_o))
    i = torch.arange(q.shape[2], device=q.device)
    gone = (i > i[:, None]) | (i < i[:, None] - left)
    P = torch.softmax((Q @ K.transpose(-1, -2) * q.shape[-1] ** -0.5).masked_fill(gone, -torch.inf), -1)
    dP = G @ V.transpose(-1, -2)
    dS = P * (dP - (P * dP).sum(-1, keepdim=True)) * q.shape[-1] ** -0.5
    return [t.permute(0, 1, 3, 2, 4) for t in (dS @ K, dS.transpose(-1, -2) @ Q, P.transpose(-1, -2) @ G)]


def _near(got, want, rows, name):
    """By norms: the one rounding of the result, which subnormal results lose bits by too, and by squares the rounding of dS (u / sqrt(3) of the norm, u =
    2^-11) and that of the o which delta is formed from, at most as much: less than u together."""
    got, want = got.double()[:, :, rows], want[:, :, rows]
    size = want.norm()
    one = float((want.to(HF).double() - want).norm() / size)
    err = float((got - want).norm() / size)
    print(f"[parity] {name}: {err:.2e}, one rounding {one:.2e}")
    assert err <= one + 2.0 ** -11, (name, err, one)


def _run(q, k, v, d_o, left):
    o, lse = mfb.window_attention_forward(q, k, v, left, 0, 0)
    return mfb.window_attention_backward(d_o, q, k, v, o, lse, left, 0, 0)


@pytest.mark.parametrize("size", [1e-4, 1e-3, 1e-2, 1.0, 1000.0])
@pytest.mark.parametrize("H,D,L,left", [(2, 64, 1500, 40), (1, 64, 2500, 1023), (2, 128, 2600, 2047), (2, 24, 900, 600)])
def test_small_gradients(H, D, L, left, size):
    q, k, v, _, d_o = (t if t is None else t.cuda() for t in base._inputs(1, 1, L, L, H, H, D, "none", HF))
    d_o = (d_o * size).to(HF)
    for name, got, want in zip(("dq", "dk"), _run(q, k, v, d_o, left), _exact(q, k, v, d_o, left)):
        _near(got, want, slice(None), name)


@pytest.mark.parametrize("D,left", [(64, 300), (128, 900)])
def test_one_large_gradient_among_small_ones(D, left):
    """The rows that do not see it are as near as they would be without it."""
    L, at = 2500, 1000
    q, k, v, _, d_o = (t.cuda() if t is not None else t for t in base._inputs(1, 1, L, L, 2, 2, D, "none", HF))
    scale = torch.full((L, 1, 1), 0.01, device="cuda")
    scale[at] = 8000
    d_o = (d_o * scale).to(HF)
    assert torch.isfinite(d_o).all()
    got, want = _run(q, k, v, d_o, left), _exact(q, k, v, d_o, left)
    others = torch.ones(L, dtype=torch.bool)
    others[at] = False
    _near(got[0], want[0], others.cuda(), "dq")
    others[at - left:at] = False
    _near(got[1], want[1], others.cuda(), "dk")
    for x, y, name in zip(got, want, ("dq", "dk", "dv")):
        assert torch.isfinite(x).all(), name
        _near(x, y, slice(None), name + " of all")

"""The operators for positions in attention at sizes where tiles, parts of lists and offsets of more than 32 bits meet."""
import pytest
import torch

import megafold_b200 as mfb
import test_window_gpu as base
from oracle import position_oracle as orc

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("B,N,Lq,Lk,H,Hk,D,left,right,sinks,mask", [
    (1, 1, 4100, 4100, 4, 2, 64, 700, 0, 4, "none"), (1, 1, 3001, 3001, 2, 1, 128, 100, 30, 130, "drop"), (2, 1, 2049, 2600, 3, 1, 32, None, 0, 0, "pad"),
    (1, 1, 1000, 3333, 8, 2, 24, 1500, 0, 65, "drop"),
])
def test_long_sequences(B, N, Lq, Lk, H, Hk, D, left, right, sinks, mask, dt):
    q, k, v, m, d_o = base._inputs(B, N, Lq, Lk, H, Hk, D, mask, dt)
    ref = orc.window(q, k, v, left, right, sinks, m, d_o, u=torch.finfo(dt).eps / 2)
    if dt == HF:
        # below 2^-14 a rounding is off by up to 2^-25 whatever the value: of each P and dS that is multiplied, and of each result
        heads = lambda t: t.double().abs().unflatten(3, (Hk, H // Hk)).sum((2, 4)).unsqueeze(2)           # noqa: E731
        for name, size in (("dq", k.double().abs().sum(2, keepdim=True).repeat_interleave(H // Hk, 3)), ("dk", heads(q)), ("dv", heads(d_o))):
            ref[name + "_tol"] = ref[name + "_tol"] + 2.0 ** -25 * (1 + size)
    c = [None if t is None else t.cuda() for t in (q, k, v, m, d_o)]
    o, lse = mfb.window_attention_forward(*c[:3], left, right, sinks, c[3])
    base._check(o, ref, "o")
    base._check(lse, ref, "lse")
    first = mfb.window_attention_backward(c[4], *c[:3], o, lse, left, right, sinks, c[3])
    again = mfb.window_attention_backward(c[4], *c[:3], o, lse, left, right, sinks, c[3])
    for name, x, y in zip(("dq", "dk", "dv"), first, again):
        base._check(x, ref, name)
        assert torch.equal(x, y), name                      # summed in a fixed order


def _room(bytes_):
    if torch.cuda.mem_get_info()[0] < bytes_:
        pytest.skip(f"needs {bytes_ / 1e9:.0f} GB")


def test_a_bias_of_more_than_32_bits_of_elements():
    """Small positions at the end of a bias and of a gradient of 2^31 + elements: those of a small bias of the same rows."""
    _room(30e9)
    B, H, L, tail = 1, 9, 15_500, 40
    assert B * H * L * L > 2 ** 31
    g = torch.Generator().manual_seed(0)
    w = torch.randn(33, H, generator=g).cuda().requires_grad_(True)
    pos = torch.cumsum(torch.randint(1, 3, (L,), generator=g), 0).cuda()
    seg = (torch.arange(L, device="cuda") // 5000)
    kw = dict(max_distance=200, scheme="log", dtype=BF)
    big = mfb.relative_position_bias(w, pos, pos, q_segments=seg, k_segments=seg, **kw)
    small = mfb.relative_position_bias(w, pos[-tail:], pos, q_segments=seg[-tail:], k_segments=seg, **kw)
    assert torch.equal(big[:, :, :, -tail:], small)
    d = torch.zeros_like(big)
    d[:, :, :, -tail:] = torch.randint(-8, 9, small.shape, generator=g).cuda()
    grad, = torch.autograd.grad(big, w, d)
    want, = torch.autograd.grad(small, w, d[:, :, :, -tail:])
    assert torch.equal(grad, want)                          # sums of small integers: exact


def test_rotation_of_more_than_32_bits_of_elements():
    """Queries of 2^31 + elements, of which the last rows are those of a small call; so are their gradients."""
    _room(40e9)
    L, H, D, tail = 131_100, 128, 128, 64
    assert L * H * D > 2 ** 31
    g = torch.Generator().manual_seed(1)
    f = (10000.0 ** (-torch.arange(64) / 64)).float().cuda()
    q, k = torch.zeros(1, 1, L, H, D, dtype=BF, device="cuda"), torch.zeros(1, 1, L, 1, D, dtype=BF, device="cuda")
    q[:, :, -tail:] = torch.randn(1, 1, tail, H, D, generator=g).cuda()
    k[:, :, -tail:] = torch.randn(1, 1, tail, 1, D, generator=g).cuda()
    pos = torch.arange(L, device="cuda")
    qo, ko = mfb.qk_norm_rotary(q.requires_grad_(True), k.requires_grad_(True), None, None, f)
    qs, ks = (t.detach()[:, :, -tail:].clone().requires_grad_(True) for t in (q, k))
    qt, kt = mfb.qk_norm_rotary(qs, ks, None, None, f, pos[-tail:])
    # the same sums in other pieces: a bit of bf16, where 24 fp32 roundings of values up to 5 (2^-17) decide over it
    near = lambda a, b: bool(((a.float() - b.float()).abs() <= 2.0 ** -7 * b.float().abs() + 2.0 ** -16).all())       # noqa: E731
    assert near(qo[:, :, -tail:], qt) and near(ko[:, :, -tail:], kt) and torch.count_nonzero(qo[:, :, :-tail]) == 0
    dq, dk = torch.zeros_like(qo), torch.zeros_like(ko)
    dq[:, :, -tail:] = torch.randn(1, 1, tail, H, D, generator=g).cuda()
    dk[:, :, -tail:] = torch.randn(1, 1, tail, 1, D, generator=g).cuda()
    a = torch.autograd.grad([qo, ko], [q, k], [dq, dk])
    b = torch.autograd.grad([qt, kt], [qs, ks], [dq[:, :, -tail:], dk[:, :, -tail:]])
    for x, y in zip(a, b):
        # a bit of bf16, and on each side 32 fp32 roundings of terms of up to 2 |d| (1 + hat^2) with |d| and hat up to 5: 2 * 32 * 2^-24 * 260
        assert bool(((x[:, :, -tail:].float() - y.float()).abs() <= 2.0 ** -7 * y.float().abs() + 2.0 ** -9.9).all())

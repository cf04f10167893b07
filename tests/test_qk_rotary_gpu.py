"""Norm and rotation of queries and keys against the definition in 64 bits."""
import pytest
import torch

import megafold_b200 as mfb
from oracle import position_oracle as orc

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
gpu = pytest.mark.gpu


def _inputs(B, N, L, H, Hk, D, R, per_head, dt, seed=0, far=False):
    g = torch.Generator().manual_seed(seed + D + L)
    q, k = torch.randn(B, N, L, H, D, generator=g).to(dt), torch.randn(B, N, L, Hk, D, generator=g).to(dt)
    qw = 1 + 0.2 * torch.randn(*((H, D) if per_head else (D,)), generator=g)
    kw = 1 + 0.2 * torch.randn(*((Hk, D) if per_head else (D,)), generator=g)
    freq = (10000.0 ** (-torch.arange(R // 2, dtype=torch.float64) * 2 / max(R, 1))).float()
    pos = torch.randint(0, 10 ** 7 if far else 500, (B, N, L), generator=g)
    dq, dk = torch.randn(q.shape, generator=g).to(dt), torch.randn(k.shape, generator=g).to(dt)
    return q, k, qw, kw, freq, pos, dq, dk


def _check(got, want, tol, what):
    err = (got.detach().double().cpu() - want).abs()
    assert (err <= tol).all(), (what, float((err / tol).max()))


def _compare(q, k, qw, kw, freq, pos, dq, dk, eps, interleaved, leaves, outs, grads):
    """The outputs are rounded once: u |x| and what 32-bit arithmetic loses, some 16 roundings of the row's values."""
    u = torch.finfo(q.dtype).eps / 2
    x = [t.double().requires_grad_(True) for t in (q, k)]
    w = [None if t is None else t.double().requires_grad_(True) for t in (qw, kw)]
    ref = [orc.rotary(x[i], w[i], freq, pos, eps, interleaved) for i in range(2)]
    names = [t for t in (*x, *w) if t is not None]
    ref_grads = torch.autograd.grad(ref, names, [dq.double(), dk.double()])
    for i in range(2):
        size = ref[i].detach().abs().amax(-1, keepdim=True)
        _check(outs[i], ref[i].detach(), u * ref[i].detach().abs() + 24 * 2.0 ** -24 * size, f"out {i}")
        # dx = rstd (w g - hat mean(w g hat)): every term is bounded by the row's largest of rstd |w g| (1 + |hat|)
        d = (dq, dk)[i].double().abs()
        rstd = 1 / torch.sqrt((x[i].detach() ** 2).mean(-1, keepdim=True) + eps)
        big = 1.0 if w[i] is None else w[i].detach().abs().max()
        hat = (x[i].detach() * rstd).abs().amax(-1, keepdim=True)
        size = rstd * big * 2 * d.amax(-1, keepdim=True) * (1 + hat * hat)
        _check(grads[i], ref_grads[i], u * ref_grads[i].abs() + 32 * 2.0 ** -24 * size, f"dx {i}")
        if w[i] is not None:
            # a sum of tokens (and heads): a rounding an addend of a thread's run, an addend is |g hat| <= 2 |d| |hat|
            size = (2 * d.amax(-1, keepdim=True) * (x[i].detach() * rstd).abs()).sum((0, 1, 2) if w[i].dim() == 2 else (0, 1, 2, 3))
            _check(grads[2 + i], ref_grads[2 + i], 2.0 ** -24 * (ref_grads[2 + i].abs() + 256 * size), f"dw {i}")


CASES = [  # B, N, L, H, Hk, D, R
    (1, 3, 17, 4, 4, 32, 32), (2, 1, 33, 16, 16, 24, 24), (1, 1, 5, 8, 2, 128, 128), (1, 1, 70, 3, 1, 64, 32), (2, 2, 9, 2, 2, 80, 80), (1, 1, 4, 2, 1, 15, 6),
    (3, 1, 1, 32, 8, 128, 128), (1, 1, 700, 1, 1, 16, 16), (1, 1, 6, 2, 2, 256, 256), (1, 1, 6, 2, 2, 251, 250), (1, 1, 3, 2, 2, 1, 0), (1, 1, 40, 2, 2, 96, 10),
    (1, 2, 8, 2, 2, 72, 40),
]


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("B,N,L,H,Hk,D,R", CASES)
def test_forward_and_backward(B, N, L, H, Hk, D, R, dt, per_head, interleaved):
    q, k, qw, kw, freq, pos, dq, dk = _inputs(B, N, L, H, Hk, D, R, per_head, dt)
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, qw, kw)]
    outs = mfb.qk_norm_rotary(*leaves, freq.cuda(), pos.cuda(), 1e-6, interleaved)
    grads = torch.autograd.grad(outs, leaves, [dq.cuda(), dk.cuda()], retain_graph=True)
    _compare(q, k, qw, kw, freq, pos, dq, dk, 1e-6, interleaved, leaves, outs, grads)
    again = torch.autograd.grad(outs, leaves, [dq.cuda(), dk.cuda()])
    assert all(torch.equal(a, b) for a, b in zip(grads, again))             # summed in a fixed order


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("B,N,L,H,Hk,D,R", [(2, 20, 131, 4, 4, 32, 32), (3, 3, 450, 5, 1, 96, 32), (2, 1, 900, 16, 4, 128, 128), (1, 4, 1100, 3, 2, 24, 8), (5, 60, 17, 4, 4, 32, 16)])
def test_positions_of_all_sequences(B, N, L, H, Hk, D, R, dt, interleaved):
    """Enough rows for the widest loads; positions of each sequence, and one set for all of them, expanded in every way or left out:
    the same numbers but for the order of the sums over tokens, which are all held to their bound."""
    q, k, qw, kw, freq, _, dq, dk = _inputs(B, N, L, H, Hk, D, R, True, dt)
    line = torch.arange(L)
    kinds = [line.expand(B, N, L).contiguous().cuda(), line.cuda(), line.cuda().int().expand(N, L), line.cuda()[None, None].expand(B, N, L), None]
    first = None
    for pos in kinds:
        leaves = [t.cuda().requires_grad_(True) for t in (q, k, qw, kw)]
        outs = mfb.qk_norm_rotary(*leaves, freq.cuda(), pos, 1e-6, interleaved)
        grads = torch.autograd.grad(outs, leaves, [dq.cuda(), dk.cuda()])
        if first is None:
            first = (*outs, *grads[:2])
            _compare(q, k, qw, kw, freq, line.expand(B, N, L), dq, dk, 1e-6, interleaved, leaves, outs, grads)
            size = [(2 * d.double().abs().amax(-1, keepdim=True) * x.double().abs() * (x.double() ** 2).mean(-1, keepdim=True).rsqrt()).sum((0, 1, 2)) for d, x in ((dq, q), (dk, k))]
            sums = grads[2:]
        assert all(torch.equal(a, b) for a, b in zip((*outs, *grads[:2]), first))
        for a, b, s in zip(grads[2:], sums, size):
            _check(a, b.double().cpu(), 2 * 2.0 ** -24 * 256 * s + 2.0 ** -23 * b.abs().double().cpu(), "dw")


@gpu
@pytest.mark.parametrize("tokens", [3000, 20011])
def test_many_tokens(tokens):
    """More tokens than threads of the backward's grid: each walks several."""
    q, k, qw, kw, freq, pos, dq, dk = _inputs(1, 1, tokens, 4, 4, 32, 32, False, BF)
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, qw, kw)]
    outs = mfb.qk_norm_rotary(*leaves, freq.cuda(), pos.cuda())
    grads = torch.autograd.grad(outs, leaves, [dq.cuda(), dk.cuda()])
    _compare(q, k, qw, kw, freq, pos, dq, dk, 1e-6, False, leaves, outs, grads)


@gpu
@pytest.mark.parametrize("dt", [FP, BF])
def test_far_positions_without_weights(dt):
    q, k, _, _, freq, pos, dq, dk = _inputs(1, 2, 40, 2, 1, 64, 64, False, dt, far=True)
    leaves = [t.cuda().requires_grad_(True) for t in (q, k)]
    outs = mfb.qk_norm_rotary(*leaves, None, None, freq.cuda(), pos.int().cuda())
    grads = torch.autograd.grad(outs, leaves, [dq.cuda(), dk.cuda()])
    _compare(q, k, None, None, freq, pos, dq, dk, 1e-6, False, leaves, outs, grads)


@gpu
def test_views_of_one_projection_default_positions_and_one_used_output():
    g = torch.Generator().manual_seed(3)
    y = torch.randn(2, 3, 20, 3 * 4 * 32, generator=g).bfloat16()
    freq = (100.0 ** (-torch.arange(16) / 16)).float()
    views = lambda t: (t[..., :128].unflatten(-1, (4, 32)), t[..., 128:256].unflatten(-1, (4, 32)))      # noqa: E731
    leaf = y.cuda().requires_grad_(True)
    w = [torch.ones(32, device="cuda", requires_grad=True) for _ in range(2)]
    qo, ko = mfb.qk_norm_rotary(*views(leaf), *w, freq.cuda())
    pos = torch.arange(20).expand(2, 3, 20)
    for got, x in zip((qo, ko), views(y)):
        want = orc.rotary(x, torch.ones(32), freq, pos, 1e-6, False)
        _check(got, want, 2.0 ** -9 * want.abs() * 2 + 24 * 2.0 ** -24 * want.abs().amax(-1, keepdim=True), "out")
    qo.sum().backward()                                                     # keys unused, gradient a broadcast view
    assert torch.count_nonzero(leaf.grad[..., 128:]) == 0 and torch.count_nonzero(leaf.grad[..., :128]) > 0
    assert torch.equal(w[1].grad, torch.zeros_like(w[1]))
    # elements that are not adjacent
    t = y[..., :128].unflatten(-1, (4, 32)).cuda()
    odd = t.transpose(-1, -2).contiguous().transpose(-1, -2)
    assert odd.stride(-1) != 1
    a = mfb.qk_norm_rotary(t, t, None, None, freq.cuda())[0]
    b = mfb.qk_norm_rotary(odd, odd, None, None, freq.cuda())[0]
    assert (a.float() - b.float()).abs().max() <= 2.0 ** -7 * a.float().abs().max()      # the same sums in another order: a bit of bf16


@gpu
def test_module_and_empty():
    m = mfb.QKNormRotary(32, num_heads=4, num_key_heads=2).cuda().bfloat16()
    assert m.inv_freq.dtype == torch.float32 and m.inv_freq.is_cuda and sorted(m.state_dict()) == ["k_weight", "q_weight"]
    q, k = torch.randn(1, 1, 8, 4, 32, device="cuda", dtype=BF), torch.randn(1, 1, 8, 2, 32, device="cuda", dtype=BF)
    qo, ko = m(q, k)
    assert qo.shape == q.shape and ko.shape == k.shape
    e = m(q[:, :, :0], k[:, :, :0])
    assert e[0].shape == (1, 1, 0, 4, 32)


def test_refusals_without_a_gpu():
    q, w, f = torch.zeros(1, 1, 4, 2, 16), torch.ones(16), torch.ones(8)
    with pytest.raises(RuntimeError, match="CUDA"):
        mfb.qk_norm_rotary(q, q, w, w, f)
    with pytest.raises(ValueError, match="pairs"):
        mfb.QKNormRotary(16, rotary_dim=18)
    import ctypes as C
    from megafold_b200 import _lib
    L = _lib.lib()
    assert L.mf_qk_rotary_fwd(None, None) == -1 and L.mf_qk_rotary_bwd(None, None) == -1
    a = _lib.QkRotaryArgs()
    assert L.mf_qk_rotary_fwd(C.byref(a), None) == -1 and L.mf_qk_rotary_bwd_workspace_bytes(C.byref(a)) == 0
    a.B = a.N = a.L = a.H = a.Hk = 1
    a.D, a.R = 257, 2
    assert L.mf_qk_rotary_fwd(C.byref(a), None) == -2
    a.D, a.R = 16, 3
    assert L.mf_qk_rotary_fwd(C.byref(a), None) == -1
    a.R, a.q_weight = 4, 16
    a.q = a.k = a.inv_freq = 16
    assert L.mf_qk_rotary_fwd(C.byref(a), None) == -1 and b"weight" in L.mf_last_error_string()


@gpu
def test_refusals():
    q, w, f = torch.zeros(1, 1, 4, 2, 16, device="cuda"), torch.ones(16, device="cuda"), torch.ones(8, device="cuda")
    for bad, kind in (((q[0], q, w, w, f), ValueError), ((q, q[:, :, :3], w, w, f), ValueError), ((q, q.half(), w, w, f), TypeError),
                      ((q, q, w, None, f), ValueError), ((q, q, w[:8], w, f), ValueError), ((q, q, w, w.half(), f), TypeError),
                      ((q, q, w, w, f.double()), TypeError), ((q, q, w, w, torch.ones(9, device="cuda")), ValueError),
                      ((q, q, w, w, f, torch.zeros(4, device="cuda")), TypeError), ((q, q, w, w, f, torch.zeros(5, device="cuda", dtype=torch.int64)), ValueError),
                      ((q, q, w, w, f.clone().requires_grad_(True)), ValueError), ((q, q, torch.ones(2, 16, device="cuda"), w, f), ValueError)):
        with pytest.raises(kind):
            mfb.qk_norm_rotary(*bad)

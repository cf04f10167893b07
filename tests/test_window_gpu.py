"""Sliding-window attention with sinks against the definition in 64 bits, element by element within the bounds of its roundings."""
import pytest
import torch

import megafold_b200 as mfb
from megafold_b200 import _lib
from oracle import position_oracle as orc

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
gpu = pytest.mark.gpu


def _inputs(B, N, Lq, Lk, H, Hk, D, mask, dt, seed=0):
    g = torch.Generator().manual_seed(seed + 31 * Lq + Lk + D)
    q, d_o = (torch.randn(B, N, Lq, H, D, generator=g).to(dt) for _ in range(2))
    k, v = (torch.randn(B, N, Lk, Hk, D, generator=g).to(dt) for _ in range(2))
    m = None
    if mask == "drop":
        m = torch.rand(B, N, 1, 1, Lk, generator=g) >= 0.2
    elif mask == "pad":
        m = torch.arange(Lk) < Lk - torch.randint(0, max(1, Lk // 2), (B, N, 1, 1, 1), generator=g)
    elif mask == "all":
        m = torch.zeros(B, 1, 1, 1, Lk, dtype=torch.bool)
    elif mask == "front":
        m = torch.arange(Lk).expand(1, N, 1, 1, Lk) >= Lk // 2
    return q, k, v, m, d_o


def _check(got, ref, name):
    want, tol = ref[name], ref[name + "_tol"]
    got = got.detach().double().cpu()
    assert got.shape == want.shape, name
    assert not got.isnan().any(), name
    same = got == want                                                      # infinite log-sum-exps
    err = torch.where(same, 0.0, (got - want).abs())
    assert (err <= tol).all(), (name, float((err / tol).max()), float(err.max()))


def _run(q, k, v, m, d_o, left, right, sinks, flags=0, back=True):
    ref = orc.window(q, k, v, left, right, sinks, m, d_o if back else None, u=torch.finfo(q.dtype).eps / 2)
    c = [None if t is None else t.cuda() for t in (q, k, v, m, d_o)]
    o, lse = mfb.window_attention_forward(*c[:3], left, right, sinks, c[3], flags)
    _check(o, ref, "o")
    _check(lse, ref, "lse")
    if back:
        grads = mfb.window_attention_backward(c[4], *c[:3], o, lse, left, right, sinks, c[3], flags)
        again = mfb.window_attention_backward(c[4], *c[:3], o, lse, left, right, sinks, c[3], flags)
        for name, x, y in zip(("dq", "dk", "dv"), grads, again):
            _check(x, ref, name)
            assert torch.equal(x, y), name                                  # summed in a fixed order
    assert _lib.lib().mf_async_status() == 0


CASES = [  # B, N, Lq, Lk, H, Hk, D, left, right, sinks, mask
    (1, 1, 1, 1, 1, 1, 8, 0, 0, 0, "none"),
    (1, 2, 64, 64, 2, 2, 32, 16, 16, 0, "none"),
    (1, 1, 65, 65, 4, 2, 32, 0, 0, 1, "none"),
    (2, 3, 130, 130, 4, 1, 24, 40, 0, 4, "drop"),
    (1, 1, 333, 333, 2, 2, 64, 64, 64, 4, "pad"),
    (1, 1, 300, 300, 8, 2, 16, None, 0, 0, "none"),
    (1, 1, 129, 129, 2, 1, 128, None, None, 0, "drop"),
    (2, 1, 700, 700, 2, 1, 64, 100, 0, 70, "pad"),
    (1, 1, 50, 500, 4, 2, 128, 127, 0, 16, "none"),
    (1, 1, 200, 1000, 2, 2, 40, 300, 20, 130, "drop"),
    (1, 1, 5, 400, 4, 4, 32, 1000, 0, 4, "pad"),
    (1, 1, 70, 20, 2, 2, 32, 8, 0, 4, "none"),            # more queries than keys: the first see none
    (1, 1, 70, 20, 2, 2, 32, 8, 60, 4, "drop"),
    (2, 2, 66, 66, 2, 2, 32, 5, 0, 0, "all"),             # nothing is kept
    (1, 2, 140, 140, 2, 2, 48, 10, 3, 9, "front"),        # rows and sinks whose keys are all masked
    (1, 1, 64, 64, 2, 2, 32, 3, 0, 1000, "none"),         # more sinks than keys
    (1, 1, 1100, 1100, 1, 1, 32, 200, 0, 4, "none"),
    (1, 1, 150, 150, 6, 2, 64, 30, 0, 4, "drop"),         # three heads share a key head: tiles of 126 and 63 rows
    (1, 2, 90, 130, 14, 2, 32, 50, 7, 3, "pad"),          # seven
    (1, 1, 40, 40, 48, 1, 16, 20, 0, 2, "none"),          # 48: two queries a tile
    (1, 1, 70, 70, 72, 1, 32, 20, 5, 2, "drop"),          # more heads than a tile has rows: one at a time
    (1, 1, 70, 300, 5, 1, 128, 100, 0, 2, "drop"),
]


@gpu
@pytest.mark.parametrize("dt", [FP, BF, HF])
@pytest.mark.parametrize("B,N,Lq,Lk,H,Hk,D,left,right,sinks,mask", CASES)
def test_forward_and_backward(B, N, Lq, Lk, H, Hk, D, left, right, sinks, mask, dt):
    _run(*_inputs(B, N, Lq, Lk, H, Hk, D, mask, dt), left, right, sinks)


@gpu
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("B,N,Lq,Lk,H,Hk,D,left,right,sinks,mask", CASES[3:9])
def test_cuda_core_kernels_on_16_bits(B, N, Lq, Lk, H, Hk, D, left, right, sinks, mask, dt):
    _run(*_inputs(B, N, Lq, Lk, H, Hk, D, mask, dt), left, right, sinks, flags=_lib.MF_FLAG_FORCE_SIMT)


@gpu
@pytest.mark.parametrize("dt", [FP, BF])
@pytest.mark.parametrize("D", [1, 7, 20, 33, 127])
def test_odd_head_sizes(D, dt):
    _run(*_inputs(1, 1, 90, 90, 2, 1, D, "drop", dt), 30, 0, 2)


@gpu
@pytest.mark.parametrize("dt", [FP, BF, HF])
@pytest.mark.parametrize("Lq,Lk", [(1, 1), (1, 63), (1, 64), (1, 65), (1, 1000), (1, 5000), (2, 3), (3, 700), (8, 129)])
@pytest.mark.parametrize("H,Hk,D", [(8, 2, 64), (8, 8, 128), (12, 1, 32), (3, 3, 24), (2, 1, 80)])
def test_few_queries(Lq, Lk, H, Hk, D, dt):
    for mask, left, sinks in (("none", 255, 4), ("drop", None, 0), ("pad", 31, 130)):
        _run(*_inputs(2, 1, Lq, Lk, H, Hk, D, mask, dt), left, 0, sinks, back=False)


@gpu
@pytest.mark.parametrize("dt", [FP, BF, HF])
@pytest.mark.parametrize("Lq,Lk", [(200, 200), (1, 300)])
def test_masked_keys_may_hold_anything(Lq, Lk, dt):
    q, k, v, m, d_o = _inputs(2, 1, Lq, Lk, 4, 2, 64, "drop", dt)
    for t, bad in ((k, float("nan")), (v, float("inf"))):
        t.masked_fill_(~m.reshape(2, 1, Lk, 1, 1), bad)
    _run(q, k, v, m, d_o, 60, 0, 4)


@gpu
@pytest.mark.parametrize("dt", [FP, BF])
def test_strided_operands_and_masks(dt):
    q, k, v, m, d_o = _inputs(2, 3, 100, 100, 2, 2, 32, "drop", dt)
    ref = orc.window(q, k, v, 30, 10, 4, m, d_o, u=torch.finfo(dt).eps / 2)
    y = torch.cat([t.flatten(3) for t in (q, k, v)], -1).cuda().requires_grad_(True)         # one projection, parts of 64
    parts = [y[..., i * 64:(i + 1) * 64].unflatten(-1, (2, 32)) for i in range(3)]
    wide = torch.zeros(2, 3, 1, 1, 200, dtype=torch.uint8)
    wide[..., ::2] = m
    o = mfb.window_attention(*parts, 30, 10, 4, wide.cuda()[..., ::2])
    _check(o, ref, "o")
    dy, = torch.autograd.grad(o, y, d_o.cuda())
    for i, name in enumerate(("dq", "dk", "dv")):
        _check(dy[..., i * 64:(i + 1) * 64].unflatten(-1, (2, 32)), ref, name)
    # heads before tokens, and elements that are not adjacent
    hl = [t.transpose(2, 3).contiguous().transpose(2, 3).cuda() for t in (q, k, v)]
    _check(mfb.window_attention(*hl, 30, 10, 4, m.cuda()), ref, "o")
    odd = [t.transpose(3, 4).contiguous().transpose(3, 4).cuda() for t in (q, k, v)]
    _check(mfb.window_attention(*odd, 30, 10, 4, m.cuda()), ref, "o")
    shifted = [torch.cat((t.flatten(), t.flatten()[:1]))[1:].cuda() for t in (q, k, v)]       # addresses off by one element
    base = [torch.empty(t.numel() + 1, dtype=dt, device="cuda") for t in (q, k, v)]
    for b, t in zip(base, (q, k, v)):
        b[1:].copy_(t.flatten())
    assert len(shifted) == 3
    _check(mfb.window_attention(*(b[1:].view(t.shape) for b, t in zip(base, (q, k, v))), 30, 10, 4, m.cuda()), ref, "o")
    # keys shared by the batch
    ke, ve = (t[:1].expand(2, 3, 100, 2, 32) for t in (k, v))
    ref = orc.window(q, ke, ve, 30, 10, 4, m, u=torch.finfo(dt).eps / 2)
    _check(mfb.window_attention(q.cuda(), k[:1].cuda().expand_as(ke), v[:1].cuda().expand_as(ve), 30, 10, 4, m.cuda()), ref, "o")


@gpu
def test_gradient_against_differences():
    q, k, v, m, d_o = _inputs(1, 1, 40, 50, 2, 1, 16, "drop", FP)
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    o = mfb.window_attention(*leaves, 9, 2, 3, m.cuda())
    grads = torch.autograd.grad(o, leaves, d_o.cuda())
    g = torch.Generator().manual_seed(5)
    for i in range(3):
        step = torch.randn(leaves[i].shape, generator=g)
        f = lambda s: (orc.window(*[(t.double() + (s * step.double() if j == i else 0)) for j, t in enumerate((q, k, v))], 9, 2, 3, m)["o"]        # noqa: E731
                       * d_o.double()).sum()
        h = 1e-5
        want = float((f(h) - f(-h)) / (2 * h))
        got = float((grads[i].cpu().double() * step.double()).sum())
        # central differences: h^2 times a third derivative of a sum of about a thousand terms, and 2^-24 of those terms
        assert abs(got - want) <= 1e-4 * float((grads[i].cpu().double() * step.double()).abs().sum()) + 1e-6


@gpu
def test_empty_lengths():
    q, k, v, _, d_o = _inputs(1, 2, 8, 8, 2, 1, 32, "none", BF)
    o, lse = mfb.window_attention_forward(q.cuda(), k[:, :, :0].cuda(), v[:, :, :0].cuda(), 4)
    assert torch.count_nonzero(o) == 0 and (lse == -float("inf")).all()
    grads = mfb.window_attention_backward(d_o.cuda(), q.cuda(), k[:, :, :0].cuda(), v[:, :, :0].cuda(), o, lse, 4)
    assert torch.count_nonzero(grads[0]) == 0 and grads[1].shape == (1, 2, 0, 1, 32)
    assert mfb.window_attention(q[:, :, :0].cuda(), k.cuda(), v.cuda(), 4).shape == (1, 2, 0, 2, 32)


def test_refusals_without_a_gpu():
    import ctypes as C
    q = torch.zeros(1, 1, 4, 2, 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        mfb.window_attention(q, q, q, 2)
    L = _lib.lib()
    assert L.mf_window_fwd(None, None) == -1 and L.mf_window_bwd(None, None) == -1 and L.mf_window_bwd_workspace_bytes(None) == 0
    a = _lib.WindowArgs()
    assert L.mf_window_fwd(C.byref(a), None) == -1
    a.B = a.N = a.Lq = a.Lk = a.H = a.Hk = a.D = 1
    a.left = -1
    assert L.mf_window_fwd(C.byref(a), None) == -1
    a.left = 0
    a.q = a.k = a.v = a.o = 16
    for field, value, status in (("D", 129, -2), ("Hk", 2, -1), ("Lk", 2 ** 30, -2), ("B", 70000, -2), ("dtype", 3, -1)):
        old = getattr(a, field)
        setattr(a, field, value)
        assert L.mf_window_fwd(C.byref(a), None) == status, field
        setattr(a, field, old)
    a.o = None
    assert L.mf_window_fwd(C.byref(a), None) == -1 and b"o must" in L.mf_last_error_string()


@gpu
def test_refusals():
    q, k = torch.zeros(1, 1, 4, 4, 16, device="cuda"), torch.zeros(1, 1, 6, 2, 16, device="cuda")
    m = torch.ones(1, 1, 1, 1, 6, dtype=torch.bool, device="cuda")
    for args, kw, kind in (((q[0], k, k, 2), {}, ValueError), ((q, k, k[:, :, :5], 2), {}, ValueError), ((q, k.half(), k, 2), {}, TypeError),
                           ((q[:, :, :, :3], k, k, 2), {}, ValueError), ((q, k, k, -1), {}, ValueError), ((q, k, k, 2), dict(sinks=-1), ValueError),
                           ((q, k, k, 2), dict(mask=m.float()), TypeError), ((q, k, k, 2), dict(mask=m[..., :5]), ValueError),
                           ((q, k, k, 2), dict(mask=m.view(1, 6)), ValueError), ((q.double(), k.double(), k.double(), 2), {}, TypeError)):
        with pytest.raises(kind):
            mfb.window_attention(*args, **kw)
    wide = torch.zeros(1, 1, 4, 2, 136, device="cuda")
    with pytest.raises(RuntimeError, match="128"):
        mfb.window_attention(wide, wide, wide, 2)
    o, lse = mfb.window_attention_forward(q, k, k, 2)
    with pytest.raises(ValueError):
        mfb.window_attention_backward(o[:, :, :2], q, k, k, o, lse, 2)
    with pytest.raises(ValueError):
        mfb.window_attention_backward(o, q, k, k, o, lse[..., :2], 2)


@gpu
@pytest.mark.parametrize("dt", [FP, BF, HF])
@pytest.mark.parametrize("Lq,Lk,left,sinks", [(1, 700, 100, 4), (90, 1000, 70, 5), (3, 300, 31, 0), (64, 700, 1, 1)])
def test_keys_that_the_window_has_passed_may_hold_anything(Lq, Lk, left, sinks, dt):
    q, k, v, m, d_o = _inputs(1, 2, Lq, Lk, 4, 2, 64, "drop", dt)
    gone = slice(sinks, Lk - Lq - left)
    ref = orc.window(q, k, v, left, 0, sinks, m, d_o, u=torch.finfo(dt).eps / 2)
    k[:, :, gone], v[:, :, gone] = float("nan"), float("inf")
    c = [t.cuda() for t in (q, k, v, m, d_o)]
    o, lse = mfb.window_attention_forward(*c[:3], left, 0, sinks, c[3])
    _check(o, ref, "o")
    _check(lse, ref, "lse")
    for name, x in zip(("dq", "dk", "dv"), mfb.window_attention_backward(c[4], *c[:3], o, lse, left, 0, sinks, c[3])):
        _check(x, ref, name)


@gpu
def test_offsets_beyond_32_bits():
    """A cache of more than 2^31 elements, of which the last query sees the end and the first keys."""
    Lk, Hk, D, left, sinks = 2_200_003, 8, 128, 300, 5
    if torch.cuda.mem_get_info()[0] < 14e9:
        pytest.skip("needs 14 GB")
    q, k, v, _, d_o = _inputs(1, 1, 2, left + 2 + sinks, 16, Hk, D, "none", BF)
    ref = orc.window(q, k, v, left, 0, sinks, None, u=2.0 ** -8)
    big = [torch.full((1, 1, Lk, Hk, D), float("nan"), dtype=BF, device="cuda") for _ in range(2)]
    for b, t in zip(big, (k, v)):
        b[:, :, :sinks], b[:, :, sinks - t.shape[2]:] = t[:, :, :sinks].cuda(), t[:, :, sinks:].cuda()
    o, lse = mfb.window_attention_forward(q.cuda(), *big, left, 0, sinks)
    _check(o, ref, "o")
    _check(lse, ref, "lse")
    small = mfb.window_attention_forward(q.cuda(), k.cuda(), v.cuda(), left, 0, sinks)
    # the same keys in other tiles: both within the bounds of the definition
    _check(small[0], ref, "o")


@gpu
@pytest.mark.parametrize("dt", [FP, BF])
def test_more_heads_of_sequences_than_a_grid_has_rows(dt):
    _run(*_inputs(1, 17000, 17, 17, 4, 4, 16, "drop", dt), 5, 0, 2)

"""Relative position bias and its gradient against the definition in 64 bits."""
import pytest
import torch

import megafold_b200 as mfb
from oracle import position_oracle as orc

pytestmark = pytest.mark.gpu

CASES = [  # B, H, Lq, Lk, rows, reach, scheme, both, segments, dtype of the table, dtype of the bias
    (1, 4, 96, 96, 65, 32, "clip", True, True, torch.float32, torch.bfloat16),
    (2, 3, 61, 61, 32, 128, "log", True, False, torch.float32, torch.float32),
    (1, 1, 1, 1, 32, 128, "log", False, False, torch.bfloat16, torch.bfloat16),
    (3, 5, 1, 777, 32, 128, "log", False, True, torch.float16, torch.float16),
    (2, 16, 7, 4096, 64, 1000, "log", True, False, torch.float32, torch.bfloat16),
    (1, 2, 130, 2056, 9, 8, "clip", False, False, torch.float32, torch.float16),
    (1, 2, 33, 70, 513, 256, "clip", True, True, torch.float32, torch.float32),
    (1, 1, 40, 3000, 1024, 16384, "log", True, False, torch.float32, torch.bfloat16),
    (4, 2, 300, 8, 4, 2, "log", True, True, torch.float32, torch.bfloat16),
]


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("B,H,Lq,Lk,count,reach,scheme,both,segments,wdt,dt", CASES)
def test_bias_and_gradient(B, H, Lq, Lk, count, reach, scheme, both, segments, wdt, dt, wide):
    g = torch.Generator().manual_seed(Lq * 7 + Lk)
    weight = torch.randn(count + segments, H, generator=g).to(wdt)
    k_pos = torch.cumsum(torch.randint(0, 1 + max(2, 2 * reach // Lk), (B, Lk), generator=g), 1) - reach
    q_pos = k_pos[:, torch.randint(0, Lk, (Lq,), generator=g)]
    q_seg, k_seg = torch.randint(0, 3, (B, Lq), generator=g), torch.randint(0, 3, (B, Lk), generator=g).sort(1).values
    d = torch.randn(B, 1, H, Lq, Lk, generator=g).to(dt)
    rows = orc.buckets(q_pos, k_pos, count, reach, scheme, both)
    if segments:
        rows = rows.masked_fill(q_seg[:, :, None] != k_seg[:, None, :], count)
    bias, grad, size = orc.relpos(weight, rows, d)

    w = weight.cuda().requires_grad_(True)
    cast = (lambda t: t.cuda()) if wide else (lambda t: t.int().cuda())
    seg = dict(q_segments=cast(q_seg), k_segments=cast(k_seg)) if segments else {}
    got = mfb.relative_position_bias(w, cast(q_pos), cast(k_pos), max_distance=reach, scheme=scheme, bidirectional=both, dtype=dt, **seg)
    assert got.shape == (B, 1, H, Lq, Lk) and got.dtype == dt
    assert torch.equal(got.detach().cpu(), bias.to(dt))                     # a look-up and one rounding
    first, = torch.autograd.grad(got, w, d.cuda(), retain_graph=True)
    # a thread's sum, a block's and the blocks': at most a rounding an addend of a thread, far below this
    u = torch.finfo(wdt).eps / 2
    assert first.dtype == wdt
    err = (first.cpu().double() - grad).abs()
    tol = u * grad.abs() + 2.0 ** -24 * 512 * size + 1e-30
    assert (err <= tol).all(), float((err / tol).max())
    again, = torch.autograd.grad(got, w, d.cuda())
    assert torch.equal(first, again)                                        # summed in a fixed order


@pytest.mark.parametrize("positions", ["none", "far away", "a gap in the keys", "a gap in the queries", "backwards", "from far to near"])
@pytest.mark.parametrize("Lk", [1, 2, 5, 9, 31, 33, 65, 70, 257, 263, 513, 1025, 1531, 2049, 2055])
@pytest.mark.parametrize("Lq", [1, 7, 300])
def test_positions_that_run_on(Lq, Lk, positions):
    """Every width of a tile around the places where columns come around its end.  The gradient's elements are small integers: all sums are exact."""
    g = torch.Generator().manual_seed(Lq + Lk)
    k, q = torch.arange(Lk), torch.arange(Lq) + Lk - Lq
    if positions == "far away":
        k, q = k + (1 << 41), q + (1 << 41)
    elif positions == "a gap in the keys":
        k = k + (k >= Lk // 2) * 3
    elif positions == "a gap in the queries":
        q = q + (torch.arange(Lq) >= Lq - Lq // 3) * 2
    elif positions == "backwards":
        k, q = -k, -q
    elif positions == "from far to near":
        q = q - (torch.arange(Lq) < Lq // 2).long() * (1 << 33)
    w = torch.zeros(24, 2, device="cuda", requires_grad=True)
    d = torch.randint(-8, 9, (1, 1, 2, Lq, Lk), generator=g)
    rows = orc.buckets(q[None], k[None], 24, 100, "log", True)
    want = torch.stack([torch.bincount(rows.flatten(), d[0, 0, h].flatten().double(), minlength=24) for h in range(2)], 1)
    args = (Lq, Lk) if positions == "none" else (q.cuda(), k.cuda())
    for dt in (torch.bfloat16, torch.float32):
        got = mfb.relative_position_bias(w, *args, max_distance=100, scheme="log", dtype=dt)
        grad, = torch.autograd.grad(got, w, d.cuda().to(dt))
        assert torch.equal(grad.cpu().double(), want)


def test_lengths_instead_of_positions_and_one_row_of_positions_for_the_batch():
    w = torch.randn(32, 3, device="cuda")
    a = mfb.relative_position_bias(w, 5, 40, max_distance=128)
    k = torch.arange(40, device="cuda")
    b = mfb.relative_position_bias(w, k[35:], k, max_distance=128)
    assert torch.equal(a, b) and a.shape == (1, 1, 3, 5, 40)
    c = mfb.relative_position_bias(w, k[35:], k.expand(2, 40), max_distance=128)
    assert torch.equal(c, b.expand(2, 1, 3, 5, 40))
    strided = torch.stack((k, k + 1), 1)[:, 0]
    assert torch.equal(mfb.relative_position_bias(w, strided[35:], strided, max_distance=128), b)


def test_far_positions_and_a_gradient_that_is_a_broadcast_view():
    w = torch.randn(32, 2, device="cuda", requires_grad=True)
    k = torch.arange(50, device="cuda") + 2 ** 40
    a = mfb.relative_position_bias(w, k, k, max_distance=128)
    assert torch.equal(a, mfb.relative_position_bias(w, 50, 50, max_distance=128))
    far = mfb.relative_position_bias(w, k[:3], torch.arange(50, device="cuda"), max_distance=128)
    assert torch.equal(far, w[15].detach().view(1, 1, 2, 1, 1).expand_as(far))
    a.sum().backward()
    rows = orc.buckets(torch.arange(50)[None], torch.arange(50)[None], 32, 128, "log", True)
    count = torch.bincount(rows.flatten(), minlength=32).float()
    assert torch.equal(w.grad.cpu(), count[:, None].expand(32, 2))          # whole numbers below 2^24: exact


def test_empty_lengths_and_refusals():
    w = torch.randn(32, 2, device="cuda", requires_grad=True)
    e = mfb.relative_position_bias(w, 0, 10, max_distance=128)
    assert e.shape == (1, 1, 2, 0, 10)
    assert torch.equal(torch.autograd.grad(e.sum(), w)[0], torch.zeros_like(w))
    k = torch.arange(8, device="cuda")
    with pytest.raises(TypeError):
        mfb.relative_position_bias(w, k.float(), k.float(), max_distance=128)
    with pytest.raises(TypeError):
        mfb.relative_position_bias(w, k.int(), k, max_distance=128)
    with pytest.raises(ValueError):
        mfb.relative_position_bias(w, k.view(1, 2, 4), k, max_distance=128)
    with pytest.raises(ValueError):
        mfb.relative_position_bias(w, k.expand(2, 8), k.expand(3, 8), max_distance=128)
    with pytest.raises(RuntimeError, match="CUDA"):
        mfb.relative_position_bias(w, k.cpu(), k.cpu(), max_distance=128)
    with pytest.raises(TypeError):
        mfb.relative_position_bias(w, k, k, max_distance=128, dtype=torch.float64)

"""The operators for positions in attention together, as a model runs them, and under what a program does around them: streams, captured
graphs, several threads."""
import threading

import pytest
import torch

import megafold_b200 as mfb
from oracle import pairformer_oracle as evo
from oracle import position_oracle as orc

pytestmark = pytest.mark.gpu
H, D, L, C = 4, 32, 72, 64


class Layer(torch.nn.Module):
    """Normed input -> q, k, v in one projection -> norm and rotation -> attention, with a learned relative bias or in a window."""

    def __init__(self, window, dtype):
        super().__init__()
        kw = dict(device="cuda", dtype=dtype)
        self.window = window
        self.qkv = mfb.LayernormLinear(C, 3 * H * D, **kw)
        self.turn = mfb.QKNormRotary(D, **kw)
        self.bias = mfb.RelativePositionBias(H, 17, 8, "clip", segments=True, device="cuda")
        with torch.no_grad():
            self.bias.weight.mul_(20)                       # values of the logits' size

    def forward(self, x, pos, seg, mask):
        q, k, v = (t.unflatten(-1, (H, D)) for t in self.qkv(x).chunk(3, -1))
        q, k = self.turn(q, k, pos[:, None])
        if self.window:
            return mfb.window_attention(q, k, v, 12, 5, 3, mask)
        return mfb.TritonEvoformer(q, k, v, mask, self.bias(pos, pos, seg, seg, dtype=x.dtype))

    def oracle(self, x, pos, seg, mask):
        """The same in 64 bits on the CPU, and the leaves its gradients belong to."""
        p = {n: t.detach().double().cpu().requires_grad_(True) for n, t in self.named_parameters()}
        xd = x.detach().double().cpu().requires_grad_(True)
        y = torch.nn.functional.layer_norm(xd, (C,), p["qkv.WEIGHT"], p["qkv.BIAS"]) @ p["qkv.linear_weight"] + p["qkv.linear_bias"]
        q, k, v = (t.unflatten(-1, (H, D)) for t in y.chunk(3, -1))
        freq, ps, m = self.turn.inv_freq.cpu(), pos.cpu(), mask.cpu()
        q, k = (orc.rotary(t, p[n], freq, ps[:, None], 1e-6, False) for t, n in ((q, "turn.q_weight"), (k, "turn.k_weight")))
        s = torch.einsum("bnihd,bnjhd->bnhij", q, k) / D ** 0.5
        if self.window:
            ok = orc.seen(L, L, 12, 5, 3)[None, None, None] & m
        else:
            rows = orc.buckets(ps, ps, 17, 8, "clip", True).masked_fill(seg.cpu()[:, :, None] != seg.cpu()[:, None], 17)
            s = s + p["bias.weight"][rows].permute(0, 3, 1, 2)[:, None]
            ok = m.expand(s.shape)
        a = torch.softmax(s.masked_fill(~ok, -1e300), -1).masked_fill(~ok, 0.0)
        return torch.einsum("bnhij,bnjhd->bnihd", a, v), {"x": xd, **p}


def _data(dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(2, 3, L, C, generator=g).to("cuda", dtype)
    pos = torch.cumsum(torch.randint(1, 3, (2, L), generator=g), 1).cuda()
    seg = (torch.arange(L) // 40).expand(2, L).contiguous().cuda()
    mask = (torch.arange(L) < torch.tensor([L, L - 9])[:, None]).view(2, 1, 1, 1, L).cuda()
    d = torch.randn(2, 3, L, H, D, generator=g).to("cuda", dtype)
    return x, pos, seg, mask, d


@pytest.mark.parametrize("window", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_a_layer_against_64_bits(window, dtype):
    torch.manual_seed(1)
    layer = Layer(window, dtype)
    x, pos, seg, mask, d = _data(dtype)
    x.requires_grad_(True)
    o = layer(x, pos, seg, mask)
    leaves = {"x": x, **dict(layer.named_parameters())}
    if window:
        leaves = {n: t for n, t in leaves.items() if not n.startswith("bias")}
    grads = torch.autograd.grad(o, list(leaves.values()), d)
    ref, ref_leaves = layer.oracle(x, pos, seg, mask)
    ref_grads = torch.autograd.grad(ref, [ref_leaves[n] for n in leaves], d.double().cpu())
    # By norms: the values pass some 16 roundings (8 tensors between the operators and, inside them, products of rounded operands, each
    # way), each off by at most u of its norm and independent of the others, so that they add by squares: 4 u, which a softmax at
    # logits of a few units passes on at most fourfold; in fp32 as many sums of some 100 addends, 16 roundings of their norm.
    u = torch.finfo(dtype).eps / 2 * (1 if dtype != torch.float32 else 16)
    for name, got, want in (("o", o, ref), *zip(leaves, grads, ref_grads)):
        err = float((got.detach().double().cpu() - want.detach()).norm() / want.detach().norm())
        print(f"[parity] {name}: {err:.2e} of {16 * u:.2e}")
        assert err <= 16 * u, (name, err)


def _graph(f, warm):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            warm()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = f()
    return g, out


@pytest.mark.parametrize("window", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_and_replayed_forward_and_backward(window, dtype):
    torch.manual_seed(2)
    layer = Layer(window, dtype)
    x, pos, seg, mask, d = _data(dtype)
    x.requires_grad_(True)
    leaves = [x, layer.qkv.linear_weight, layer.turn.q_weight] + ([] if window else [layer.bias.weight])

    def step():
        o = layer(x, pos, seg, mask)
        return [o.detach(), *torch.autograd.grad(o, leaves, d)]

    # (no eager graph of the same leaves may live through the capture: torch then leaves the captured stream)
    first, got1 = _graph(step, step)
    second, got2 = _graph(step, step)                      # two graphs, replayed one after the other
    for seed in (3, 4):
        x2, pos2, seg2, _, d2 = _data(dtype, seed)
        with torch.no_grad():
            for a, b in ((x, x2), (pos, pos2), (seg, seg2), (d, d2)):
                a.copy_(b)
        first.replay()
        second.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, got1, got2))


def test_a_few_queries_captured():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(2, 1, n, h, 64, generator=g).bfloat16().cuda() for n, h in ((1, 8), (900, 2), (900, 2)))
    with torch.no_grad():
        graph, o = _graph(lambda: mfb.window_attention(q, k, v, 500, 0, 4), lambda: mfb.window_attention(q, k, v, 500, 0, 4))
        q.copy_(torch.randn(q.shape, generator=g))
        graph.replay()
        assert torch.equal(o, mfb.window_attention(q, k, v, 500, 0, 4))


def test_side_streams_and_threads():
    """Calls from several threads on streams of their own, with different inputs, give what they give alone."""
    layers = [Layer(w, torch.bfloat16) for w in (False, True)]
    data = [_data(torch.bfloat16, s) for s in range(4)]

    def step(i):
        x, pos, seg, mask, d = data[i]
        x = x.detach().requires_grad_(True)
        o = layers[i % 2](x, pos, seg, mask)
        return [o.detach(), *torch.autograd.grad(o, [x, layers[i % 2].qkv.linear_weight], d)]

    want = [step(i) for i in range(4)]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(10):
                got[i] = step(i)
        s.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(4):
        # the projection's weight gradient is a sum in arrival order, which differs in the last bits
        assert torch.equal(want[i][0], got[i][0])
        assert (want[i][1].float() - got[i][1].float()).norm() <= 2.0 ** -8 * want[i][1].float().norm()


def test_changed_inputs_are_noticed():
    """An input changed in place between forward and backward is an error, as everywhere in torch."""
    x, pos, seg, mask, d = _data(torch.bfloat16)
    w = torch.randn(18, H, device="cuda", requires_grad=True)
    b = mfb.relative_position_bias(w, pos, pos, max_distance=8, scheme="clip", q_segments=seg, k_segments=seg)
    pos.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        b.sum().backward()


def test_no_forward_mode_and_no_transforms():
    w = torch.randn(32, 2, device="cuda")
    q = torch.randn(1, 1, 8, 2, 16, device="cuda")
    f = torch.ones(8, device="cuda")
    for call, arg in ((lambda t: mfb.relative_position_bias(t, 4, 4, max_distance=128), w), (lambda t: mfb.window_attention(t, t, t, 3), q),
                      (lambda t: mfb.qk_norm_rotary(t, t, None, None, f)[0], q)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.jvp(call, (arg,), (arg,))
        with torch.no_grad(), pytest.raises((RuntimeError, NotImplementedError)):
            with torch.autograd.forward_ad.dual_level():
                call(torch.autograd.forward_ad.make_dual(arg, arg))


def test_gradients_against_differences():
    g = torch.Generator().manual_seed(4)
    # the table: the result is linear in it, so that a difference is the gradient's product up to the rounding of sums of 900 terms
    w, d = torch.randn(16, 2, generator=g), torch.randn(1, 1, 2, 30, 30, generator=g)
    step = torch.randn(16, 2, generator=g)
    leaf = w.cuda().requires_grad_(True)
    grad, = torch.autograd.grad(mfb.relative_position_bias(leaf, 30, 30, max_distance=20), leaf, d.cuda())
    pos = torch.arange(30)[None]
    f = lambda t: float((orc.relpos(t, orc.buckets(pos, pos, 16, 20, "log", True))[0] * d.double()).sum())        # noqa: E731
    want = f(w.double() + step.double()) - f(w.double())
    assert abs(float((grad.cpu().double() * step.double()).sum()) - want) <= 1e-5 * float((grad.cpu().double() * step.double()).abs().sum())
    # norm and rotation: central differences of a function whose values are sums of some 1000 terms of size one
    q, k = torch.randn(1, 1, 9, 3, 24, generator=g), torch.randn(1, 1, 9, 1, 24, generator=g)
    qw, kw = 1 + 0.2 * torch.randn(24, generator=g), 1 + 0.2 * torch.randn(24, generator=g)
    freq, pos = torch.rand(8, generator=g), torch.arange(9)
    dq, dk = torch.randn(q.shape, generator=g), torch.randn(k.shape, generator=g)
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, qw, kw)]
    outs = mfb.qk_norm_rotary(*leaves, freq.cuda(), pos.cuda(), 1e-6, True)
    grads = torch.autograd.grad(outs, leaves, [dq.cuda(), dk.cuda()])
    for i in range(4):
        step = torch.randn(leaves[i].shape, generator=g).double()

        def value(h):
            a = [t.double() + (h * step if j == i else 0) for j, t in enumerate((q, k, qw, kw))]
            return float((orc.rotary(a[0], a[2], freq, pos, 1e-6, True) * dq.double()).sum() + (orc.rotary(a[1], a[3], freq, pos, 1e-6, True) * dk.double()).sum())

        want = (value(1e-5) - value(-1e-5)) / 2e-5
        prod = grads[i].cpu().double() * step
        assert abs(float(prod.sum()) - want) <= 1e-5 * float(prod.abs().sum()) + 1e-6, i


def test_evo_oracle_is_the_plain_softmax():
    """The attention oracle of the older tests and the one above agree (so that the layer's test rests on both)."""
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(1, 2, 9, 2, 8, generator=g) for _ in range(3))
    m, b = torch.ones(1, 2, 1, 1, 9, dtype=torch.bool), torch.zeros(1, 1, 2, 9, 9)
    assert torch.allclose(evo.evo_attention(q, k, v, m, b).double(), orc.window(q, k, v, None, None, 0)["o"], atol=1e-5)

"""Positions in attention: three operators of the package, each with its plain form and its definition in 64 bits.

A case is a dict of plain values; ``kind`` says which operator it goes through.

* ``relpos``: a pair bias ``[B, 1, H, Lq, Lk]`` looked up in a learned table by the bucket of the distance of two positions,
  with the gradient of the table.
* ``rotary``: RMS norm of every head of queries and keys, and the rotation by their positions, in one pass, with its backward.
* ``window``: attention that sees a window around the query's position and the first few tokens (sinks), with its backward and,
  for a few queries on a long row of keys, its single-token form.

The sizes are those of this repository's crops (384 and 768 tokens, 4 heads of 32, 16 heads of 24) and generic ones.
``run`` computes the plain form, or, where ``own`` is true, calls the package.
"""
import math
from fractions import Fraction

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


def listed():
    return [
        # the learned relative position encoding of a training crop: residue distances clipped to 32, one more bucket for
        # another chain, as a bf16 pair bias of the triangle attention's four heads; parameters in fp32
        dict(name="relpos_chains_384", kind="relpos", B=1, H=4, Lq=384, Lk=384, scheme="clip", buckets=65, max_distance=32, bidirectional=True,
             segments=True, dtype="bf16", train=True),
        # logarithmic buckets over a long sequence when predicting, sixteen heads: the largest bias
        dict(name="relpos_log_4096", kind="relpos", B=1, H=16, Lq=4096, Lk=4096, scheme="log", buckets=32, max_distance=128, bidirectional=True,
             segments=False, dtype="bf16", train=False),
        # one more training size, a batch of two at an odd length with a table and a bias in fp32
        dict(name="relpos_log_1531_fp32", kind="relpos", B=2, H=8, Lq=1531, Lk=1531, scheme="log", buckets=64, max_distance=800, bidirectional=True,
             segments=False, dtype="fp32", train=True),
        # one new token against the keys before it, causal buckets: latency only
        dict(name="relpos_step_8191", kind="relpos", B=8, H=16, Lq=1, Lk=8191, scheme="log", buckets=32, max_distance=128, bidirectional=False,
             segments=False, dtype="fp16", train=False),
        # queries and keys of triangle attention at crop 384, in training
        dict(name="rotary_triangle_384", kind="rotary", B=1, N=384, L=384, H=4, Hk=4, D=32, R=32, interleaved=False, per_head=False, far=False,
             dtype="bf16", train=True),
        # one new token of each of 32 sequences, grouped heads of 128, positions up to a million: latency only
        dict(name="rotary_step_32", kind="rotary", B=32, N=1, L=1, H=32, Hk=8, D=128, R=128, interleaved=False, per_head=False, far=True, dtype="bf16",
             train=False),
        # sixteen heads of 24 at a ragged length, a weight for every head, interleaved pairs on a part of each head, fp32
        dict(name="rotary_single_777_fp32", kind="rotary", B=2, N=1, L=777, H=16, Hk=16, D=24, R=16, interleaved=True, per_head=True, far=False,
             dtype="fp32", train=True),
        # atoms of a structure in training: a window to both sides, four memory tokens in front that every atom sees
        dict(name="window_atoms_4603", kind="window", B=1, N=1, Lq=4603, Lk=4603, H=4, Hk=4, D=32, left=64, right=64, sinks=4, mask="pad", dtype="bf16",
             train=True),
        # a parity check or a debugging run in fp32 at an odd size, keys dropped at random
        dict(name="window_single_517_fp32", kind="window", B=2, N=1, Lq=517, Lk=517, H=8, Hk=2, D=24, left=100, right=0, sinks=3, mask="drop",
             dtype="fp32", train=True),
        # one new token of each of 64 sequences on its cached keys, grouped heads: the single-token form
        dict(name="window_step_64", kind="window", B=64, N=1, Lq=1, Lk=4100, H=32, Hk=8, D=128, left=1023, right=0, sinks=4, mask="pad", dtype="bf16",
             train=False),
        # a chunk of a long prompt behind the tokens before it, heads of 128
        dict(name="window_chunk_2048", kind="window", B=2, N=1, Lq=2048, Lk=6001, H=16, Hk=4, D=128, left=2047, right=0, sinks=16, mask="none",
             dtype="fp16", train=False),
        # a long training sequence with grouped heads: the largest
        dict(name="window_long_16384", kind="window", B=1, N=1, Lq=16384, Lk=16384, H=16, Hk=4, D=64, left=1023, right=0, sinks=4, mask="none",
             dtype="bf16", train=True),
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the listed ones' ranges that costs no more than the largest of them."""
    most = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    while True:
        case = _draw(rng)
        if all(work(case)[k] <= most[k] for k in most):
            return case


def _draw(rng):
    kind = rng.choice(["relpos", "rotary", "window", "window"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "relpos":
        scheme = rng.choice(["clip", "log"])
        B, H = rng.choice([1, 1, 2, 4]), _log_int(rng, 1, 16)
        train = rng.random() < 0.5
        if rng.random() < 0.3:
            Lq, Lk = _log_int(rng, 1, 8), _log_int(rng, 64, 16384)
            train = False
        else:
            Lq = Lk = _log_int(rng, 48, 2048)
        if scheme == "clip":
            r = _log_int(rng, 8, 64)
            buckets, reach, both = 2 * r + 1, r, True
        else:
            both = rng.random() < 0.6
            buckets, reach = 2 * _log_int(rng, 8, 32), _log_int(rng, 64, 1024)
        return dict(kind=kind, B=B, H=H, Lq=Lq, Lk=Lk, scheme=scheme, buckets=buckets, max_distance=reach, bidirectional=both,
                    segments=rng.random() < 0.4, dtype=dtype, train=train)
    if kind == "rotary":
        D = rng.choice([16, 24, 32, 64, 80, 96, 128])
        R = D if rng.random() < 0.7 else 2 * rng.randint(1, D // 2)
        sort = rng.choice(["step", "pair", "single"])
        train = sort != "step" and rng.random() < 0.7
        if sort == "step":
            B, N, L, H, Hk = _log_int(rng, 1, 256), 1, 1, 32, rng.choice([4, 8, 32])
        elif sort == "pair":
            L = _log_int(rng, 48, 384)
            B, N, H, Hk, D = 1, L, 4, 4, 32
            R = min(R, D)
        else:
            B, N, L, H = rng.choice([1, 2]), 1, _log_int(rng, 32, 4096), rng.choice([4, 8, 16])
            Hk = rng.choice([1, H // 2, H])
        return dict(kind=kind, B=B, N=N, L=L, H=H, Hk=Hk, D=D, R=R, interleaved=rng.random() < 0.4, per_head=rng.random() < 0.4,
                    far=rng.random() < 0.3, dtype=dtype, train=train)
    mask = rng.choice(["pad", "drop", "none", "none"])
    sort = rng.choice(["step", "chunk", "train", "train"])
    D = rng.choice([16, 24, 32, 64, 64, 128])
    Hk = rng.choice([1, 2, 4])
    H = Hk * rng.choice([1, 1, 2, 4, 8])
    sinks = rng.choice([0, 1, 4, 64, 130])
    left = _log_int(rng, 1, 2048)
    right = rng.choice([0, 0, left, rng.randint(0, left)])
    if sort == "step":
        return dict(kind=kind, B=_log_int(rng, 1, 64), N=1, Lq=rng.choice([1, 1, 1, 2, 5]), Lk=_log_int(rng, 5, 16384), H=H, Hk=Hk, D=D, left=left,
                    right=0, sinks=sinks, mask=mask, dtype=dtype, train=False)
    if sort == "chunk":
        Lq = _log_int(rng, 16, 2048)
        return dict(kind=kind, B=rng.choice([1, 2]), N=1, Lq=Lq, Lk=Lq + _log_int(rng, 1, 6000), H=H, Hk=Hk, D=D, left=left, right=right, sinks=sinks,
                    mask=mask, dtype=dtype, train=rng.random() < 0.3)
    L = _log_int(rng, 1, 4096)
    N = _log_int(rng, 1, 16) if L <= 512 else 1
    return dict(kind=kind, B=rng.choice([1, 2]), N=N, Lq=L, Lk=L, H=H, Hk=Hk, D=D, left=left, right=right, sinks=sinks, mask=mask, dtype=dtype,
                train=True)


# ---------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    randn = lambda *s: torch.randn(*s, device="cuda", generator=g)                                        # noqa: E731
    randint = lambda lo, hi, *s: torch.randint(lo, hi, s, device="cuda", generator=g)                     # noqa: E731
    state = dict(case=case)
    if case["kind"] == "relpos":
        B, H, Lq, Lk = (case[x] for x in ("B", "H", "Lq", "Lk"))
        weight = 0.5 * randn(case["buckets"] + case["segments"], H)
        if not case["train"]:
            weight = weight.to(dt)
        # residue numbers that run on with gaps now and then, from anywhere; the queries are the last of the keys
        k_pos = torch.cumsum(1 + 7 * (torch.rand(B, Lk, device="cuda", generator=g) < 0.01), 1) + randint(0, 1000, B, 1)
        state.update(weight=weight, k_pos=k_pos, q_pos=k_pos[:, Lk - Lq:].contiguous())
        if case["segments"]:
            k_seg = torch.cumsum((torch.rand(B, Lk, device="cuda", generator=g) < 4 / Lk).long(), 1)
            state.update(k_seg=k_seg, q_seg=k_seg[:, Lk - Lq:].contiguous())
        if case["train"]:
            weight.requires_grad_(True)
            state["d_out"] = randn(B, 1, H, Lq, Lk).to(dt)
        return state
    B, N, D = case["B"], case["N"], case["D"]
    if case["kind"] == "rotary":
        L, H, Hk, R = case["L"], case["H"], case["Hk"], case["R"]
        # queries and keys are parts of one projection, as they leave it
        both = randn(B, N, L, H + Hk, D).to(dt)
        q, k = both[..., :H, :], both[..., H:, :]
        q_weight = 1 + 0.1 * randn(*((H, D) if case["per_head"] else (D,)))
        k_weight = 1 + 0.1 * randn(*((Hk, D) if case["per_head"] else (D,)))
        inv_freq = 10000.0 ** (-torch.arange(R // 2, device="cuda", dtype=torch.float64) * 2 / R)
        positions = torch.arange(L, device="cuda") + randint(0, 1_000_000 if case["far"] else 64, B, N, 1)
        state.update(q=q, k=k, q_weight=q_weight, k_weight=k_weight, inv_freq=inv_freq.float(), positions=positions)
        if case["train"]:
            q, k = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
            q_weight.requires_grad_(True)
            k_weight.requires_grad_(True)
            state.update(q=q, k=k, d_out=(randn(B, N, L, H, D).to(dt), randn(B, N, L, Hk, D).to(dt)))
        return state
    Lq, Lk, H, Hk = case["Lq"], case["Lk"], case["H"], case["Hk"]
    q, k, v = randn(B, N, Lq, H, D).to(dt), randn(B, N, Lk, Hk, D).to(dt), randn(B, N, Lk, Hk, D).to(dt)
    mask = None
    if case["mask"] == "drop":
        mask = torch.rand(B, N, 1, 1, Lk, device="cuda", generator=g) >= 0.1
    elif case["mask"] == "pad":
        mask = torch.arange(Lk, device="cuda") < Lk - randint(0, max(1, Lk // 12), B, N, 1, 1, 1)
    state.update(q=q, k=k, v=v, mask=mask)
    if case["train"]:
        for t in (q, k, v):
            t.requires_grad_(True)
        state["d_out"] = randn(B, N, Lq, H, D).to(dt)
    return state


# ------------------------------------------------------------------------------------------------------------- one pass
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"relpos": _own_relpos, "rotary": _own_rotary, "window": _own_window}[kind](state)
    with torch.no_grad():
        return {"relpos": _plain_relpos, "rotary": _plain_rotary, "window": _plain_window}[kind](state)


def _own_relpos(s):
    import megafold_b200 as mfb
    c = s["case"]
    bias = mfb.relative_position_bias(s["weight"], s["q_pos"], s["k_pos"], max_distance=c["max_distance"], scheme=c["scheme"],
                                      bidirectional=c["bidirectional"], q_segments=s.get("q_seg"), k_segments=s.get("k_seg"), dtype=DTYPES[c["dtype"]])
    if not c["train"]:
        return [bias]
    return [bias.detach(), *torch.autograd.grad(bias, s["weight"], s["d_out"])]


def _own_rotary(s):
    import megafold_b200 as mfb
    c = s["case"]
    out = mfb.qk_norm_rotary(s["q"], s["k"], s["q_weight"], s["k_weight"], s["inv_freq"], s["positions"], eps=1e-6, interleaved=c["interleaved"])
    if not c["train"]:
        return list(out)
    return [*(t.detach() for t in out), *torch.autograd.grad(out, (s["q"], s["k"], s["q_weight"], s["k_weight"]), s["d_out"])]


def _own_window(s):
    import megafold_b200 as mfb
    c = s["case"]
    o = mfb.window_attention(s["q"], s["k"], s["v"], left=c["left"], right=c["right"], sinks=c["sinks"], mask=s["mask"])
    if not c["train"]:
        return [o]
    return [o.detach(), *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["d_out"])]


# ---- plain forms ---------------------------------------------------------------------------------------------------
def _plain_buckets(c, q_pos, k_pos):
    """Bucket of every pair, [B, Lq, Lk]."""
    d = k_pos[:, None, :] - q_pos[:, :, None]
    reach, count = c["max_distance"], c["buckets"]
    if c["scheme"] == "clip":
        return d.clamp(-reach, reach) + reach
    side = 0
    if c["bidirectional"]:
        count //= 2
        side = torch.where(d > 0, count, 0)
        n = d.abs()
    else:
        n = (-d).clamp(min=0)
    near = count // 2
    t = torch.log(n.clamp(min=near).double() / near) / math.log(reach / near) * (count - near)
    whole = torch.round(t)
    t = torch.where((t - whole).abs() < 1e-9, whole, torch.floor(t))                 # a distance that lies on a border
    return side + torch.where(n < near, n, (near + t.long()).clamp(max=count - 1))


def _plain_relpos(s):
    c = s["case"]
    dt = DTYPES[c["dtype"]]
    bucket = _plain_buckets(c, s["q_pos"], s["k_pos"])
    if c["segments"]:
        bucket = torch.where(s["q_seg"][:, :, None] == s["k_seg"][:, None, :], bucket, c["buckets"])
    w = s["weight"].float()
    bias = w.T[:, bucket].transpose(0, 1).to(dt)[:, None]
    if not c["train"]:
        return [bias]
    d = s["d_out"][:, 0].float()
    rows = [torch.where((bucket == b)[:, None], d, 0.0).sum((0, 2, 3), dtype=torch.float64) for b in range(w.shape[0])]
    return [bias, torch.stack(rows).to(s["weight"].dtype)]


def _turn(x, cos, sin, R, interleaved, back=False):
    """The rotation of the first R elements of each head; ``back``: its transpose."""
    if back:
        sin = -sin
    if interleaved:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., R:]), -1)


def _plain_rotary(s):
    c = s["case"]
    angle = s["positions"].double()[..., None, None] * s["inv_freq"].double()
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    outs, grads, weights = [], [], []
    for i, (x, w) in enumerate(((s["q"], s["q_weight"]), (s["k"], s["k_weight"]))):
        x32 = x.float()
        rstd = torch.rsqrt((x32 * x32).mean(-1, keepdim=True) + 1e-6)
        hat = x32 * rstd
        outs.append(_turn(hat * w, cos, sin, c["R"], c["interleaved"]).to(x.dtype))
        if c["train"]:
            g = _turn(s["d_out"][i].float(), cos, sin, c["R"], c["interleaved"], back=True)
            gw = g * w
            grads.append((rstd * (gw - hat * (gw * hat).mean(-1, keepdim=True))).to(x.dtype))
            weights.append((g * hat).sum((0, 1, 2) if w.dim() == 2 else (0, 1, 2, 3), dtype=torch.float64).to(w.dtype))
    return outs + grads + weights


def _plain_window(s):
    c = s["case"]
    left, right, sinks = c["left"], c["right"], c["sinks"]
    q, k, v, mask = s["q"], s["k"], s["v"], s["mask"]
    B, N, Lq, H, D = q.shape
    Lk, Hk = k.shape[2], k.shape[3]
    dev, scale = q.device, D ** -0.5
    heads = lambda t: t.float().permute(0, 1, 3, 2, 4)                                                    # noqa: E731
    qf, kf, vf = heads(q).reshape(B, N, Hk, H // Hk, Lq, D), heads(k).unsqueeze(3), heads(v).unsqueeze(3)
    keep = torch.ones(B, N, Lk, dtype=torch.bool, device=dev) if mask is None else mask.expand(B, N, 1, 1, Lk).reshape(B, N, Lk)
    o = torch.empty_like(qf)
    if c["train"]:
        do = heads(s["d_out"]).reshape(B, N, Hk, H // Hk, Lq, D)
        dq, dk, dv = torch.empty_like(qf), torch.zeros_like(kf), torch.zeros_like(vf)
    step = 512
    for i0 in range(0, Lq, step):
        i1 = min(Lq, i0 + step)
        p = torch.arange(i0, i1, device=dev) + (Lk - Lq)
        lo = min(Lk, max(0, i0 + Lk - Lq - left))
        hi = min(Lk, max(lo, i1 + Lk - Lq + right))
        spans = [(lo, hi)] if min(sinks, lo) == 0 else [(0, min(sinks, lo)), (lo, hi)]
        pick = lambda t, dim: torch.cat([t.narrow(dim, a, b - a) for a, b in spans], dim)                 # noqa: E731
        j = torch.cat([torch.arange(a, b, device=dev) for a, b in spans])
        seen = (j <= p[:, None] + right) & ((j >= p[:, None] - left) | (j < sinks))
        seen = seen & pick(keep, 2)[:, :, None, None, None, :]
        kc, vc = pick(kf, 4), pick(vf, 4)
        x = (qf[..., i0:i1, :] @ kc.transpose(-1, -2)) * scale
        x = torch.where(seen, x, -math.inf)
        top = x.amax(-1, keepdim=True) if x.shape[-1] else x.new_full((*x.shape[:-1], 1), -math.inf)
        e = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
        total = e.sum(-1, keepdim=True)
        e = e / torch.where(total == 0, 1.0, total)
        oc = e @ vc
        o[..., i0:i1, :] = oc
        if c["train"]:
            dc = do[..., i0:i1, :]
            ds = e * (dc @ vc.transpose(-1, -2) - (dc * oc).sum(-1, keepdim=True)) * scale
            dq[..., i0:i1, :] = ds @ kc
            dkc = (ds.transpose(-1, -2) @ qf[..., i0:i1, :]).sum(3, keepdim=True)
            dvc = (e.transpose(-1, -2) @ dc).sum(3, keepdim=True)
            at = 0
            for a, b in spans:
                dk[..., a:b, :] += dkc[..., at:at + b - a, :]
                dv[..., a:b, :] += dvc[..., at:at + b - a, :]
                at += b - a
    tokens = lambda t: t.flatten(2, 3).permute(0, 1, 3, 2, 4).to(q.dtype).contiguous()                    # noqa: E731
    return [tokens(t) for t in ((o, dq, dk, dv) if c["train"] else (o,))]


# ---- definitions in 64 bits ------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"relpos": _exact_relpos, "rotary": _exact_rotary, "window": _exact_window}[case["kind"]](s)


def _exact_relpos(s):
    c = s["case"]
    reach, count = c["max_distance"], c["buckets"]
    far = reach + 1
    table = np.zeros(2 * far + 1, dtype=np.int64)                  # bucket of each distance from -far to far; beyond: as at the end
    for d in range(-far, far + 1):
        if c["scheme"] == "clip":
            table[d + far] = min(max(d, -reach), reach) + reach
            continue
        half = count // 2 if c["bidirectional"] else count
        n = abs(d) if c["bidirectional"] else max(-d, 0)
        near = half // 2
        if n < near:
            b = n
        else:
            # the largest b with (n / near) ^ (half - near) >= (reach / near) ^ (b - near), in whole numbers
            ratio, top, b = Fraction(n, near) ** (half - near), Fraction(reach, near), near
            while b < half - 1 and ratio >= top ** (b + 1 - near):
                b += 1
        table[d + far] = b + (half if c["bidirectional"] and d > 0 else 0)
    d = (s["k_pos"].unsqueeze(1) - s["q_pos"].unsqueeze(2)).clamp(-far, far) + far
    bucket = torch.from_numpy(table).cuda()[d]
    if c["segments"]:
        bucket[s["q_seg"].unsqueeze(2) != s["k_seg"].unsqueeze(1)] = count
    w = s["weight"].double()
    bias = torch.stack([w[:, h][bucket] for h in range(w.shape[1])], 1).unsqueeze(1)
    if not c["train"]:
        return [bias]
    order = bucket.flatten().argsort(stable=True)
    sizes = torch.bincount(bucket.flatten(), minlength=w.shape[0]).tolist()
    grad = torch.zeros_like(w)
    for h in range(w.shape[1]):
        for b, part in enumerate(s["d_out"][:, 0, h].double().flatten()[order].split(sizes)):
            grad[b, h] = part.sum()
    return [bias, grad]


def _exact_rotary(s):
    c = s["case"]
    R, D = c["R"], c["D"]
    first = torch.arange(R // 2, device="cuda") * (2 if c["interleaved"] else 1)
    second = first + (1 if c["interleaved"] else R // 2)
    z = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["positions"].double()[..., None, None] * s["inv_freq"].double())
    outs, leaves = [], []
    for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
        x, w = x.detach().double(), w.detach().double()
        if c["train"]:
            x.requires_grad_(True)
            w.requires_grad_(True)
        leaves.append((x, w))
        with torch.enable_grad():
            y = x / torch.sqrt(torch.square(x).sum(-1, keepdim=True) / D + 1e-6) * w
            pair = torch.complex(y[..., first], y[..., second]) * z
            out = y.clone()
            out[..., first], out[..., second] = pair.real, pair.imag
        outs.append(out)
    if not c["train"]:
        return outs
    (q, qw), (k, kw) = leaves
    grads = torch.autograd.grad(outs, (q, k, qw, kw), [d.double() for d in s["d_out"]])
    return [*(t.detach() for t in outs), *grads]


def _exact_window(s):
    c = s["case"]
    q, k, v = (s[x].detach().double() for x in "qkv")
    B, N, Lq, H, D = q.shape
    Lk, Hk = k.shape[2], k.shape[3]
    out = [torch.zeros_like(q)]
    if c["train"]:
        out += [torch.zeros_like(t) for t in (q, k, v)]
        d_out = s["d_out"].double()
    j = torch.arange(Lk, device="cuda")
    rows = max(1, 40_000_000 // max(1, Lk))
    for b in range(B):
        for n in range(N):
            keep = torch.ones(Lk, dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"].expand(B, N, 1, 1, Lk)[b, n, 0, 0]
            for i in range(0, Lq, rows):
                at = slice(i, min(Lq, i + rows))
                p = (torch.arange(Lq, device="cuda")[at] + Lk - Lq).unsqueeze(1)
                hidden = ~((j <= p + c["right"]) & ((j >= p - c["left"]) | (j < c["sinks"])) & keep)
                for h in range(H):
                    kh, vh = k[b, n, :, h * Hk // H], v[b, n, :, h * Hk // H]
                    x = torch.mm(q[b, n, at, h], kh.T).div_(math.sqrt(D)).masked_fill_(hidden, -math.inf)
                    x = torch.nan_to_num_(torch.softmax(x, 1), nan=0.0)              # a row that sees nothing
                    oh = x @ vh
                    out[0][b, n, at, h] = oh
                    if c["train"]:
                        gh = d_out[b, n, at, h]
                        out[3][b, n, :, h * Hk // H] += x.T @ gh
                        x *= gh @ vh.T - (gh * oh).sum(1, keepdim=True)
                        x /= math.sqrt(D)
                        out[1][b, n, at, h] = x @ kh
                        out[2][b, n, :, h * Hk // H] += x.T @ q[b, n, at, h]
    return out


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    es = SIZE[case["dtype"]]
    if case["kind"] == "relpos":
        pairs = case["B"] * case["H"] * case["Lq"] * case["Lk"]
        table = (case["buckets"] + case["segments"]) * case["H"] * (4 if case["train"] else es)
        return {"bytes": (2 if case["train"] else 1) * (pairs * es + table) + 8 * case["B"] * (case["Lq"] + case["Lk"]) * (1 + case["segments"]),
                "flops": pairs if case["train"] else 0}
    if case["kind"] == "rotary":
        tokens = case["B"] * case["N"] * case["L"]
        n = tokens * (case["H"] + case["Hk"]) * case["D"]
        return {"bytes": n * es * (4 if case["train"] else 2) + 8 * tokens, "flops": n * (18 if case["train"] else 7)}
    B, N, Lq, Lk, H, Hk, D = (case[x] for x in ("B", "N", "Lq", "Lk", "H", "Hk", "D"))
    p = np.arange(Lq) + Lk - Lq
    hi = np.clip(p + case["right"] + 1, 0, Lk)
    lo = np.clip(p - case["left"], 0, hi)
    pairs = int((hi - lo + np.minimum(np.minimum(case["sinks"], hi), lo)).sum())
    cover = np.zeros(Lk + 1, dtype=np.int64)
    np.add.at(cover, lo, 1)
    np.add.at(cover, hi, -1)
    used = np.cumsum(cover[:-1]) > 0
    used[:min(case["sinks"], int(hi.max(initial=0)))] = True
    rows_q, rows_k = B * N * Lq * H * D, B * N * int(used.sum()) * Hk * D
    moved = 2 * rows_q + 2 * rows_k
    if case["train"]:
        moved += 2 * rows_q + 2 * B * N * Lk * Hk * D            # d_out and dq, dk and dv; the second reading of q, k and v is no need
    if case["mask"] != "none":
        moved_mask = B * N * int(used.sum())
    else:
        moved_mask = 0
    return {"bytes": moved * es + moved_mask, "flops": B * N * H * pairs * D * (14 if case["train"] else 4)}

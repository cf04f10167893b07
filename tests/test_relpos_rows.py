"""Tables of relative positions up to the largest, in one direction and in two."""
import ctypes as C

import pytest
import torch

import megafold_b200 as mfb
from megafold_b200 import _lib
from megafold_b200.relative_position import _buckets
from oracle import position_oracle as orc

CASES = [  # rows, reach, scheme, both: the last ones of a direction have more borders than half a table
    (513, 512, "clip", False), (514, 513, "clip", False), (1024, 1023, "clip", False), (1023, 511, "clip", True),
    (513, 900, "log", False), (514, 2000, "log", False), (1024, 16384, "log", False), (1024, 16384, "log", True),
]


@pytest.mark.parametrize("count,reach,scheme,both", CASES)
def test_borders(count, reach, scheme, both):
    edges, rows = _buckets(count, reach, scheme, both)
    assert list(edges) == sorted(edges) and edges[-1] <= reach
    for d in {s * (e + x) for e in (*edges[:3], *edges[len(edges) // 2:][:3], *edges[-3:], reach, 10 ** 6) for x in (-1, 0, 1) for s in (-1, 1)}:
        m = sum(e <= abs(d) for e in edges)
        assert (rows[0] + rows[1] * m if d > 0 else rows[2] + rows[3] * m) == orc.bucket(d, count, reach, scheme, both), d


def test_tables_beyond_the_limit_are_refused_where_they_are_made():
    assert mfb.RelativePositionBias(2, 1024, 16384, "log", False).weight.shape == (1024, 2)
    assert mfb.RelativePositionBias(2, 1023, 511, "clip", segments=True).weight.shape == (1024, 2)
    for kw in (dict(num_buckets=1025, max_distance=16384, bidirectional=False), dict(num_buckets=1024, max_distance=16384, segments=True),
               dict(num_buckets=1026, max_distance=16384)):
        with pytest.raises(ValueError, match="1024"):
            mfb.RelativePositionBias(2, **kw)


def test_the_library_takes_the_borders_of_the_largest_table():
    L = _lib.lib()
    a = _lib.RelposArgs()
    a.B = a.H = a.Lq = a.Lk = 1
    a.rows, a.n_edges, a.edges = 1024, 1023, (C.c_int32 * 1023)(*range(1, 1024))
    assert L.mf_relpos_fwd(C.byref(a), None) == -1 and b"weight and bias" in L.mf_last_error_string()         # what is still missing
    a.n_edges, a.edges = 1024, (C.c_int32 * 1024)(*range(1, 1025))
    assert L.mf_relpos_fwd(C.byref(a), None) == -2 and b"1023" in L.mf_last_error_string()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("Lq,Lk", [(1, 2500), (150, 1301)])
@pytest.mark.parametrize("count,reach,scheme,both", CASES)
def test_bias_and_gradient(count, reach, scheme, both, Lq, Lk, dt):
    """The gradient's elements are small integers: all sums are exact."""
    g = torch.Generator().manual_seed(count + Lq)
    k = torch.cumsum(torch.randint(1, 2 + 2 * reach // Lk, (1, Lk), generator=g), 1)
    q = k[:, -Lq:]
    rows = orc.buckets(q, k, count, reach, scheme, both)
    weight = torch.randn(count, 2, generator=g)
    d = torch.randint(-8, 9, (1, 1, 2, Lq, Lk), generator=g)
    w = weight.cuda().requires_grad_(True)
    got = mfb.relative_position_bias(w, q.cuda(), k.cuda(), max_distance=reach, scheme=scheme, bidirectional=both, dtype=dt)
    assert torch.equal(got.detach().cpu(), orc.relpos(weight, rows).to(dt))
    grad, = torch.autograd.grad(got, w, d.cuda().to(dt))
    want = torch.stack([torch.bincount(rows.flatten(), d[0, 0, h].flatten().double(), minlength=count) for h in range(2)], 1)
    assert torch.equal(grad.cpu().double(), want)

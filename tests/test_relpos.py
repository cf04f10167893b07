"""Buckets of relative positions against their definition, and what the operator refuses (no GPU needed)."""
import pytest
import torch

import megafold_b200 as mfb
from megafold_b200.relative_position import _buckets
from oracle import position_oracle as orc


def _row(edges, rows, d):
    m = sum(e <= abs(d) for e in edges)
    return rows[0] + rows[1] * m if d > 0 else rows[2] + rows[3] * m


@pytest.mark.parametrize("count,reach,scheme,both", [
    (65, 32, "clip", True), (9, 8, "clip", False), (32, 128, "log", True), (32, 128, "log", False), (64, 800, "log", True), (16, 16, "log", True),
    (4, 2, "log", True), (2, 16384, "log", False), (6, 5, "log", True), (512, 16384, "log", True),
])
def test_buckets_are_the_definition(count, reach, scheme, both):
    edges, rows = _buckets(count, reach, scheme, both)
    assert list(edges) == sorted(edges) and edges[-1] <= reach
    span = list(range(-300, 301)) + [-reach - 1, -reach, -reach + 1, reach - 1, reach, reach + 1, 10 ** 6, -10 ** 6]
    span += [s * (e + x) for e in edges[-40:] for x in (-1, 0, 1) for s in (-1, 1)]
    for d in span:
        assert _row(edges, rows, d) == orc.bucket(d, count, reach, scheme, both), d
        assert 0 <= _row(edges, rows, d) < count


def test_a_distance_on_a_border_enters_the_next_bucket():
    # 8 small buckets, then 8 up to 128: each border is 8 * 16^(k / 8), and 8 * 16^(1/4) = 16 is a whole number
    edges, rows = _buckets(32, 128, "log", True)
    assert 16 in edges and _row(edges, rows, -15) == 9 and _row(edges, rows, -16) == 10


@pytest.mark.parametrize("count,reach,scheme,both,what", [
    (64, 32, "clip", True, "buckets"), (33, 128, "log", True, "even"), (32, 8, "log", True, "logarithmic"), (32, 0, "log", True, "max_distance"),
    (32, 16385, "log", True, "max_distance"), (32, 128, "linear", True, "scheme"), (1, 128, "log", False, "logarithmic"),
])
def test_bad_buckets_are_refused(count, reach, scheme, both, what):
    with pytest.raises(ValueError, match=what):
        mfb.RelativePositionBias(4, count, reach, scheme, both)


def test_refusals_without_a_gpu():
    w = torch.zeros(32, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        mfb.relative_position_bias(w, 4, 8, max_distance=128)
    with pytest.raises(ValueError, match="rows, heads"):
        mfb.relative_position_bias(w[0], 4, 8, max_distance=128)
    with pytest.raises(ValueError, match="1024"):
        mfb.relative_position_bias(torch.zeros(1025, 2), 4, 8, max_distance=2048)
    with pytest.raises(TypeError, match="two"):
        mfb.relative_position_bias(w, torch.arange(4), 8, max_distance=128)
    m = mfb.RelativePositionBias(2, segments=True)
    assert m.weight.shape == (33, 2) and sorted(m.state_dict()) == ["weight"]
    with pytest.raises(ValueError, match="segments"):
        m(4, 8)


def test_bad_arguments_are_refused_by_the_library():
    import ctypes as C
    from megafold_b200 import _lib
    L = _lib.lib()
    assert L.mf_relpos_fwd(None, None) == -1 and L.mf_relpos_bwd(None, None) == -1 and L.mf_relpos_bwd_workspace_bytes(None) == 0
    a = _lib.RelposArgs()
    assert L.mf_relpos_fwd(C.byref(a), None) == -1
    a.B = a.H = a.Lq = a.Lk = 1
    a.rows = 5
    a.n_edges, a.edges = 2, (C.c_int32 * 2)(3, 2)
    assert L.mf_relpos_fwd(C.byref(a), None) == -1 and b"ascending" in L.mf_last_error_string()
    a.edges = (C.c_int32 * 2)(3, 20000)
    assert L.mf_relpos_fwd(C.byref(a), None) == -1
    a.edges = (C.c_int32 * 2)(2, 3)
    a.rows = 1025
    assert L.mf_relpos_fwd(C.byref(a), None) == -2
    a.rows = 5
    a.q_pos = 16
    assert L.mf_relpos_fwd(C.byref(a), None) == -1 and b"positions" in L.mf_last_error_string()

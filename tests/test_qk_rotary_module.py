"""QKNormRotary built without memory first (the meta device) and given memory later, as large models are."""
import pytest
import torch

import megafold_b200 as mfb

ARGS = [dict(head_dim=32), dict(head_dim=128, rotary_dim=64, base=500000.0), dict(head_dim=24, rotary_dim=0), dict(head_dim=16, num_heads=4, num_key_heads=2)]


def _meta(kw):
    with torch.device("meta"):
        return mfb.QKNormRotary(**kw)


@pytest.mark.parametrize("kw", ARGS)
def test_memory_given_by_to_empty(kw):
    want = mfb.QKNormRotary(**kw)
    with torch.device("meta"):                              # memory is given where it is named
        m = torch.nn.Sequential(mfb.QKNormRotary(**kw)).to_empty(device="cpu")[0]
    assert torch.equal(m.inv_freq, want.inv_freq) and m.inv_freq.dtype == torch.float32
    with torch.no_grad():
        want.q_weight.fill_(3)
        want.k_weight.fill_(5)
    m.load_state_dict(want.state_dict())
    assert torch.equal(m.q_weight, want.q_weight) and torch.equal(m.k_weight, want.k_weight)
    m.reset_parameters()
    assert torch.equal(m.q_weight, torch.ones_like(m.q_weight)) and torch.equal(m.k_weight, torch.ones_like(m.k_weight))
    m.bfloat16()
    assert m.q_weight.dtype == torch.bfloat16 and torch.equal(m.inv_freq, want.inv_freq)


@pytest.mark.parametrize("kw", ARGS)
def test_memory_given_by_the_state_dict(kw):
    want = mfb.QKNormRotary(**kw)
    m = _meta(kw)
    m.load_state_dict(want.state_dict(), assign=True)
    m = torch.nn.Sequential(m).to("cpu")[0]
    assert torch.equal(m.inv_freq, want.inv_freq)


def test_without_memory_it_stays_so_and_other_frequencies_are_kept():
    m = _meta(dict(head_dim=32)).half()
    assert m.inv_freq.is_meta and m.inv_freq.dtype == torch.float32
    m = mfb.QKNormRotary(32)
    m.inv_freq.mul_(0.25)                                   # positions of a longer row
    want = m.inv_freq.clone()
    assert torch.equal(m.double().inv_freq, want)
    m.to("meta")
    assert m.inv_freq.is_meta

"""Sizes beyond 32 bits are refused, not cut down to what is left of them."""
import pytest
import torch

import megafold_b200 as mfb

pytestmark = pytest.mark.gpu
FAR = 2 ** 32 + 8          # 8 in 32 bits


@pytest.mark.parametrize("axis", [0, 1, 2])
def test_more_tokens_than_32_bits_hold(axis):
    x = torch.ones(1, 1, 1, 1, 1, dtype=torch.bfloat16, device="cuda")
    q = x.expand(*(FAR if i == axis else 1 for i in range(5)))
    f = torch.empty(0, device="cuda")
    for leaf in (q, q.detach().requires_grad_(True)):
        with pytest.raises(RuntimeError, match="tokens"):
            mfb.qk_norm_rotary(leaf, leaf, None, None, f)
    two = x.expand(2 ** 16, 2 ** 15, 1, 1, 1)               # 2^31 tokens in two dimensions
    with pytest.raises(RuntimeError, match="tokens"):
        mfb.qk_norm_rotary(two, two, None, None, f)


def test_more_heads_or_elements_than_32_bits_hold():
    x = torch.ones(1, 1, 1, 1, 1, dtype=torch.bfloat16, device="cuda")
    f = torch.empty(0, device="cuda")
    q = x.expand(1, 1, 1, FAR, 1)
    for args in ((q, x), (x, q), (q, q)):
        with pytest.raises(RuntimeError, match="heads"):
            mfb.qk_norm_rotary(*args, None, None, f)
    q = x.expand(1, 1, 1, 1, FAR)
    with pytest.raises(RuntimeError, match="head size"):
        mfb.qk_norm_rotary(q, q, None, None, f)


def test_more_batch_elements_than_32_bits_hold():
    w = torch.zeros(32, 1, dtype=torch.bfloat16, device="cuda")
    pos = torch.zeros(1, 1, dtype=torch.int64, device="cuda").expand(FAR, 1)
    for weight in (w, w.clone().requires_grad_(True)):
        with pytest.raises(RuntimeError, match="65535"):
            mfb.relative_position_bias(weight, pos, pos, max_distance=128)
    x = torch.ones(1, 1, 1, 1, 1, dtype=torch.bfloat16, device="cuda")
    for axis in (0, 1, 2, 3):
        q = x.expand(*(FAR if i == axis else n for i, n in enumerate(x.shape)))
        with pytest.raises(RuntimeError, match="not supported|exceeds|above"):
            mfb.window_attention(q, q, q, 4)

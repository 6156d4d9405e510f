"""Heads past what the selective scan takes, up to more than 32 bits hold."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def policy(gpu):
    from navi_amd import policy

    return policy


def test_more_heads_than_numbers_of_32_bits(policy):
    heads = (1 << 32) + 4
    one = torch.zeros(1, 1, 1, 8, device="cuda")
    x, dt, a = one.expand(1, 1, heads, 8), one[..., 0].expand(1, 1, heads), torch.empty(heads, device="cuda")
    state = torch.empty(1, 1, 8, 8, device="cuda").expand(1, heads, 8, 8)
    for heads in (heads, 16385):
        with pytest.raises(RuntimeError, match="heads must be at most 16384"):
            policy.selective_scan(x[:, :, :heads], dt[..., :heads], a[:heads], one, one)
        with pytest.raises(RuntimeError, match="heads must be at most 16384"):
            policy.selective_scan_step(x[:, 0, :heads], dt[:, 0, :heads], a[:heads], one[:, 0], one[:, 0], state[:, :heads])

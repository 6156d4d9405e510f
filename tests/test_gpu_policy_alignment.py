"""Outputs at any element's address (``navi_amd.policy`` through its C entry points): what PyTorch's
allocator never gives, a caller from C may."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def policy(gpu):
    from navi_amd import policy

    return policy


@pytest.mark.parametrize("dim", [64, 36, 33])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("first", [1, 2, 3])
def test_rollouts_into_any_address(policy, first, dtype, dim):
    gen = torch.Generator(device="cuda").manual_seed(4)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    q, k = (torch.nn.functional.normalize(rand(2, 70, 2, 32), dim=-1).to(dtype) for _ in range(2))
    v, g, beta = rand(2, 70, 2, dim).to(dtype), -rand(2, 70, 2).abs(), torch.sigmoid(rand(2, 70, 2))
    want = policy.gated_delta_rule(q, k, v, g, beta)
    flat = torch.full((v.numel() + 8,), 7.0, dtype=dtype, device="cuda")
    out = flat[first:first + v.numel()].view(v.shape)
    matrices = torch.empty((4, 2, policy._native.CHUNK_MATRICES), device="cuda")
    rule = policy._pack_rule(q, k, v, g, beta, None, 32 ** -0.5, None, out, None, matrices)
    policy._call(policy._native.lib().navi_delta_forward, q.device, rule)
    assert torch.equal(out, want)
    assert (flat[:first] == 7.0).all() and (flat[first + v.numel():] == 7.0).all()

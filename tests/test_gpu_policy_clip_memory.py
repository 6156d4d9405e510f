"""``clip_grad_norm`` (``navi_amd.policy``) and tensors that share memory or lie next to each other."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def policy(gpu):
    from navi_amd import policy

    return policy


def test_a_tensor_named_twice_is_refused(policy):
    g, h = torch.ones(100000, device="cuda"), torch.ones(7, device="cuda")
    for grads in ([g, g], [g, h, g.view(100, 1000)], [g, g[99999:]]):
        with pytest.raises(RuntimeError, match="share memory"):
            policy.clip_grad_norm(grads, 1.0)
        assert torch.equal(g, torch.ones_like(g)) and torch.equal(h, torch.ones_like(h))
    one = torch.empty_like(g)
    with pytest.raises(RuntimeError, match="share memory"):
        policy.clip_grad_norm([g, g.clone()], 1.0, out=[one, one])
    with pytest.raises(RuntimeError, match="share memory"):
        policy.clip_grad_norm([g[:-1]], 1.0, out=[g[1:]])


def test_what_shares_no_written_memory_runs(policy):
    flat = torch.full((4096,), 2.0, device="cuda")
    parts = [flat[:1], flat[1:100], flat[1000:], flat[100:1000]]  # next to each other, in any order
    norm = policy.clip_grad_norm(parts, 1.0)
    assert abs(float(norm) - 128.0) <= 1e-4
    assert torch.allclose(flat, torch.full_like(flat, 2.0 / 128.0))
    g = torch.ones(64, device="cuda")  # read twice, written to two places
    out = [torch.zeros_like(g) for _ in range(2)]
    norm = policy.clip_grad_norm([g, g], 1.0, out=out)
    assert abs(float(norm) - 128.0 ** 0.5) <= 1e-5
    assert torch.equal(out[0], out[1]) and torch.equal(g, torch.ones_like(g))
    empty = torch.empty(0, device="cuda")
    policy.clip_grad_norm([empty, empty, g], 1.0)

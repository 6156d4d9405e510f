"""Steps of the gated delta rule (``navi_amd.policy``) whose output shares memory with an input."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def policy(gpu):
    from navi_amd import policy

    return policy


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("envs, heads, dim", [(1, 1, 5), (3, 2, 64), (700, 2, 96)])
def test_steps_into_their_values_and_next_to_their_inputs(policy, envs, heads, dim, dtype):
    gen = torch.Generator(device="cuda").manual_seed(2)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    packed = rand(4, envs, heads, dim).to(dtype)  # queries, keys, values and outputs next to each other
    packed[:2] = torch.nn.functional.normalize(packed[:2].float(), dim=-1).to(dtype)
    q, k, v, out = packed
    g, beta, state = -rand(envs, heads).abs(), torch.sigmoid(rand(envs, heads)), rand(envs, heads, dim, dim)
    states = [state.clone() for _ in range(4)]
    want = policy.gated_delta_step(q, k, v, g, beta, states[0])
    assert torch.equal(policy.gated_delta_step(q, k, v, g, beta, states[1], out=out), want)
    for bad in (q, k):
        with pytest.raises(RuntimeError, match="shares memory"):
            policy.gated_delta_step(q, k, v, g, beta, states[3], out=bad)
    assert torch.equal(policy.gated_delta_step(q, k, v, g, beta, states[2], out=v), want)  # in place
    assert torch.equal(v, want)
    assert torch.equal(states[1], states[0]) and torch.equal(states[2], states[0]) and torch.equal(states[3], state)

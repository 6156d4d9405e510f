"""The policy's operators (``navi_amd.policy``) and autograd: writes that it is told of."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def policy(gpu):
    from navi_amd import policy

    return policy


def frame(envs=3, heads=2, dim=32, dtype=torch.float32, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    x = [torch.nn.functional.normalize(rand(envs, heads, dim), dim=-1).to(dtype) for _ in range(2)]
    x += [rand(envs, heads, dim).to(dtype), -rand(envs, heads).abs(), torch.sigmoid(rand(envs, heads))]
    return x, rand(envs, heads, dim, dim)


# ---- writes ----


def test_a_step_into_a_saved_output_is_an_error_backward(policy):
    x, state = frame()
    weight = torch.randn(32, 8, device="cuda", requires_grad=True)
    out = torch.empty_like(x[2])
    policy.gated_delta_step(*x, state, out=out)
    y = out @ weight  # (saves out for the weight's gradient)
    version = out._version
    policy.gated_delta_step(*x, state, out=out)
    assert out._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_a_step_of_a_saved_state_is_an_error_backward(policy):
    x, state = frame()
    weight = torch.randn(32, device="cuda", requires_grad=True)
    y = (state * weight).sum()
    policy.gated_delta_step(*x, state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_an_output_that_requires_grad_is_refused(policy):
    x, state = frame()
    kept = state.clone()
    for out in (torch.empty_like(x[2]).requires_grad_(), torch.empty_like(x[2]).requires_grad_() * 2):
        with pytest.raises(RuntimeError, match="no gradients"):
            policy.gated_delta_step(*x, state, out=out)
        assert torch.equal(state, kept)
        with torch.no_grad():
            policy.gated_delta_step(*x, state.clone(), out=out)


def test_inference_tensors(policy):
    with torch.inference_mode():
        x, state = frame()
        out = torch.empty_like(x[2])
        policy.gated_delta_step(*x, state, out=out)
        policy.clip_grad_norm([out], 1.0)
    assert torch.isfinite(out).all()

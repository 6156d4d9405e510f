"""The policy's operators (``navi_amd.policy``) and autograd: writes that it is told of, derivatives
that they do not have."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

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


def rollout(envs=2, steps=130, heads=2, dim=32, dtype=torch.float32, seed=0):
    x, state = frame(envs * steps, heads, dim, dtype, seed)
    return [t.unflatten(0, (envs, steps)) for t in x], state[:envs].clone()


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


# ---- derivatives that the operators do not have ----


@pytest.mark.parametrize("dual", range(6))
def test_forward_mode_is_refused(policy, dual):
    x, state = frame()
    short, long = rollout(steps=3), rollout()
    with forward_ad.dual_level():
        with_tangent = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for given, carried in ((x, state), short, long):
            args = list(given)
            if dual < 5:
                args[dual] = with_tangent(args[dual])
            else:
                carried = with_tangent(carried)
            with pytest.raises(RuntimeError, match="forward-mode"):
                if given is x:
                    policy.gated_delta_step(*args, carried)
                else:
                    policy.gated_delta_rule(*args, initial_state=carried)
        policy.gated_delta_step(*x, state)  # (none of its own inputs is one)
        policy.gated_delta_rule(*long[0], initial_state=long[1])


@pytest.mark.parametrize("dual", ["q", "k", "q_weight", "k_weight", "cos", "sin"])
def test_forward_mode_of_norms_is_refused(policy, dual):
    gen = torch.Generator(device="cuda").manual_seed(1)
    args = {n: torch.randn(2, 3, 1, 32, generator=gen, device="cuda") for n in ("q", "k")}
    args |= {n: torch.ones(32, device="cuda") for n in ("q_weight", "k_weight")}
    args |= {n: torch.ones(3, 8, device="cuda") for n in ("cos", "sin")}
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            policy.qk_norm(**{**args, dual: forward_ad.make_dual(args[dual], torch.ones_like(args[dual]))})
        policy.qk_norm(**args)


def test_forward_mode_of_clipping_is_refused(policy):
    g = torch.ones(5, device="cuda")
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            policy.clip_grad_norm([forward_ad.make_dual(g, torch.ones_like(g))], 1.0)
        with pytest.raises(RuntimeError, match="forward-mode"):
            policy.clip_grad_norm([g], 1.0, out=[forward_ad.make_dual(g.clone(), torch.ones_like(g))])


@pytest.mark.parametrize("name", ["cos", "sin"])
def test_tables_that_require_grad_are_refused(policy, name):
    q = torch.randn(2, 3, 1, 32, device="cuda")
    args = {n: torch.ones(3, 8, device="cuda").requires_grad_(n == name) for n in ("cos", "sin")}
    with pytest.raises(RuntimeError, match="cos and sin have no gradients"):
        policy.qk_norm(q, q, **args)
    with torch.no_grad():
        policy.qk_norm(q, q, **args)

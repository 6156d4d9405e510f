"""The policy's operators (``navi_amd.policy``) and autograd: writes that it is told of, derivatives
that they do not have, gradients of some of the inputs, streams and threads."""

from __future__ import annotations

import threading

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


# ---- gradients ----


@pytest.mark.parametrize("wanted", [[0], [1], [2], [3], [4], [5], [0, 3], [2, 5]], ids=str)
@pytest.mark.parametrize("steps", [3, 130])
def test_gradients_of_some_inputs(policy, steps, wanted):
    """The same numbers, whichever inputs they are asked for."""
    x, state = rollout(steps=steps)
    inputs = [*x, state]
    run = lambda args: policy.gated_delta_rule(*args[:5], initial_state=args[5], return_state=True)  # noqa: E731
    all_of = [t.clone().requires_grad_() for t in inputs]
    o, final = run(all_of)
    grads = [torch.randn_like(o), torch.randn_like(final)]
    want = torch.autograd.grad([o, final], all_of, grads)
    some = [t.clone().requires_grad_(i in wanted) for i, t in enumerate(inputs)]
    o, final = run(some)
    got = torch.autograd.grad([o, final], [some[i] for i in wanted], grads)
    for i, g in zip(wanted, got):
        assert torch.equal(g, want[i])


def test_a_shared_gates_gradient_is_the_sum_over_heads(policy):
    x, _ = rollout(heads=4)
    gate, beta = (t[:, :, :1].clone().requires_grad_() for t in x[3:])
    o = policy.gated_delta_rule(*x[:3], gate.expand(2, 130, 4), beta.expand(2, 130, 4))
    whole = [t.detach().expand(2, 130, 4).contiguous().requires_grad_() for t in (gate, beta)]
    want = policy.gated_delta_rule(*x[:3], *whole)
    assert torch.equal(o, want)
    grad = torch.randn_like(o)
    got = torch.autograd.grad(o, [gate, beta], grad)
    for a, b in zip(got, torch.autograd.grad(want, whole, grad)):
        # (four numbers summed in float32: three roundings of partial sums)
        assert ((a.double() - b.double().sum(-1, keepdim=True)).abs() <= 3 * 2.0 ** -24 * b.abs().sum(-1, keepdim=True)).all()
        assert float(b.abs().max()) > 0


# ---- streams and threads ----


def test_two_streams_on_inputs_of_their_own(policy):
    given = [rollout(envs=6, steps=700, dim=64, dtype=torch.bfloat16, seed=s) for s in (1, 2)]
    want = [policy.gated_delta_rule(*x, initial_state=s) for x, s in given]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in given], [[], []]
    for _ in range(4):
        for i, (x, s) in enumerate(given):
            with torch.cuda.stream(streams[i]):
                got[i].append(policy.gated_delta_rule(*x, initial_state=s))
    for i, stream in enumerate(streams):
        stream.synchronize()
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_two_threads(policy):
    given = [rollout(envs=4, steps=200, seed=s) for s in (3, 4)]

    def once(i):
        x, state = given[i]
        leaves = [t.clone().requires_grad_() for t in x]
        o = policy.gated_delta_rule(*leaves, initial_state=state)
        q, k = policy.qk_norm(x[0], x[1])
        return [o, q, k, *torch.autograd.grad(o, leaves, torch.ones_like(o))]

    want = [once(i) for i in range(2)]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got = once(i)
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                        wrong.append(i)
        except Exception as error:  # noqa: BLE001 (told to the test's own thread)
            wrong.append(error)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong

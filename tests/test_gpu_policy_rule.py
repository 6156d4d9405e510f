"""The gated delta rule (``navi_amd.policy``) on the GPU against the recurrence in float64.

Tolerances. Products run on exact splits of float32 and accumulate in float32, so an output
is a sum of some hundred terms with relative errors of a few 2^-24 each, which the triangle's
inverse may enlarge a few times: 32 x 2^-24 of the output's norm for float32 values, and the
output's own rounding on top where it is of 16 bits. The gradient of g is a
difference of terms that the gradient of beta, times beta, stands for: 64 x 2^-24 of both.
"""

from __future__ import annotations

import math

import pytest
import torch

from . import policy_reference as ref

pytestmark = pytest.mark.gpu

TOL = 32 * ref.EPS


@pytest.fixture(scope="module")
def policy(gpu):
    from navi_amd import policy

    return policy


def make(envs, steps, hk, hv, kd, vd, dtype, seed=0, alike=0.6):
    gen = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    unit = lambda x: torch.nn.functional.normalize(x, dim=-1)  # noqa: E731
    x = {"q": unit(rand(envs, steps, hk, kd)).to(dtype),
         "k": unit(rand(envs, steps, hk, kd) + alike * rand(envs, 1, hk, kd)).to(dtype),
         "v": rand(envs, steps, hv, vd).to(dtype),
         "g": -torch.exp(rand(envs, steps, hv) * 1.5 - 3.0),
         "beta": torch.sigmoid(rand(envs, steps, hv) + 0.5)}
    state = 0.3 * rand(envs, hv, kd, vd)
    starts = torch.rand(envs, steps, generator=gen) < 0.04
    return {k: v.cuda() for k, v in x.items()}, state.cuda(), starts.cuda()


def tolerance(dtype, base=TOL):
    return base + (ref.ROUNDING[dtype] if dtype != torch.float32 else 0.0)


SIZES = [
    (1, 1, 1, 1, 1, 1, torch.float32),
    (2, 1, 1, 2, 64, 64, torch.bfloat16),
    (3, 15, 1, 1, 16, 16, torch.float32),
    (2, 63, 2, 2, 64, 64, torch.float16),
    (2, 64, 1, 1, 64, 64, torch.float32),
    (1, 65, 1, 3, 33, 17, torch.float32),
    (2, 128, 2, 2, 64, 256, torch.bfloat16),
    (1, 129, 2, 4, 100, 72, torch.float16),
    (1, 130, 1, 1, 128, 130, torch.float32),
    (1, 257, 1, 2, 128, 128, torch.bfloat16),
    (5, 70, 3, 3, 7, 5, torch.bfloat16),
]


@pytest.mark.parametrize("with_state", [False, True])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_rule_and_gradients(policy, size, with_state):
    dtype = size[-1]
    x, state, starts = make(*size)
    if not with_state:
        state = starts = None
    given = list(x) + (["state"] if with_state else [])
    leaves = {n: t.clone().requires_grad_() for n, t in x.items()}
    if with_state:
        leaves["state"] = state.clone().requires_grad_()
    got = policy.gated_delta_rule(*[leaves[n] for n in x], starts=starts, initial_state=leaves.get("state"),
                                  return_state=with_state)
    o, final = got if with_state else (got, None)

    scale = size[4] ** -0.5
    exact = {n: t.detach().cpu().double().requires_grad_() for n, t in leaves.items()}
    want_o, want_final = ref.rule(*[exact[n] for n in x], starts, exact.get("state"), scale)
    assert ref.off(o, want_o) <= tolerance(dtype)
    gen = torch.Generator().manual_seed(9)
    grads = [torch.randn(o.shape, generator=gen).to(dtype)]
    outs, want_outs = [o], [want_o]
    if with_state:
        assert ref.off(final, want_final) <= TOL
        grads.append(torch.randn(final.shape, generator=gen))
        outs.append(final)
        want_outs.append(want_final)
    back = dict(zip(given, torch.autograd.grad(outs, [leaves[n] for n in given], [t.cuda() for t in grads])))
    want = dict(zip(given, torch.autograd.grad(want_outs, [exact[n] for n in given], [t.double() for t in grads])))
    for n in ("q", "k", "v"):
        assert back[n].dtype == dtype
        assert ref.off(back[n], want[n]) <= tolerance(dtype), n
    assert ref.off(back["beta"], want["beta"]) <= 2 * TOL
    room = 2 * TOL * float(want["g"].norm() + (want["beta"] * exact["beta"].detach()).norm())
    assert float((back["g"].cpu().double() - want["g"]).norm()) <= room
    if with_state:
        assert ref.off(back["state"], want["state"]) <= TOL
        assert torch.equal(back["g"].cpu()[starts.cpu()], torch.zeros_like(back["g"].cpu()[starts.cpu()]))


@pytest.mark.parametrize("steps", [1, 2, 4, 5])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_short_rollouts_without_gradients(policy, steps, dtype):
    x, state, starts = make(3, 6, 2, 4, 50, 36, dtype, seed=steps)
    starts = torch.rand(starts.shape, device="cuda") < 0.3
    x = {n: t[:, 1:1 + steps] for n, t in x.items()}  # (views)
    x["q"] = x["q"][:, :1].expand(x["q"].shape)
    o, final = policy.gated_delta_rule(*x.values(), starts=starts[:, 1:1 + steps], initial_state=state, return_state=True)
    want_o, want_final = ref.rule(*x.values(), starts[:, 1:1 + steps], state, 50 ** -0.5)
    assert ref.off(o, want_o) <= tolerance(dtype)
    assert ref.off(final, want_final) <= TOL
    o = policy.gated_delta_rule(*x.values())
    assert ref.off(o, ref.rule(*x.values(), None, None, 50 ** -0.5)[0]) <= tolerance(dtype)


LONG = [  # few heads and many chunks: walked in segments that are joined
    (1, 64 * 8, 1, 1, 64, 64, torch.float32),
    (1, 64 * 9 + 5, 1, 2, 33, 70, torch.bfloat16),
    (2, 64 * 12 + 1, 1, 2, 128, 128, torch.float16),
    (1, 64 * 21 + 63, 1, 1, 100, 150, torch.float32),
    (8, 64 * 39 + 1, 4, 8, 10, 12, torch.bfloat16),  # (workgroups of five segments: more than one to a CU)
]


@pytest.mark.parametrize("ends", [True, False], ids=["episodes", "one episode"])
@pytest.mark.parametrize("size", LONG, ids=str)
def test_long_walks(policy, size, ends):
    dtype = size[-1]
    x, state, starts = make(*size, seed=21)
    starts = (torch.rand(starts.shape, device="cuda") < 0.003) if ends else None
    x["g"] *= 0.05  # (a state that lasts through segments)
    leaves = [t.clone().requires_grad_() for t in x.values()]
    s0 = state.clone().requires_grad_()
    o, final = policy.gated_delta_rule(*leaves, starts=starts, initial_state=s0, return_state=True)
    exact = [t.detach().cpu().double().requires_grad_() for t in leaves]
    e0 = state.cpu().double().requires_grad_()
    want_o, want_final = ref.rule(*exact, starts, e0, size[4] ** -0.5)
    assert ref.off(o, want_o) <= tolerance(dtype)
    assert ref.off(final, want_final) <= TOL
    gen = torch.Generator().manual_seed(5)
    go, gs = torch.randn(o.shape, generator=gen).to(dtype), torch.randn(final.shape, generator=gen)
    back = torch.autograd.grad([o, final], leaves + [s0], [go.cuda(), gs.cuda()])
    want = torch.autograd.grad([want_o, want_final], exact + [e0], [go.double(), gs.double()])
    for a, b in zip(back[:3], want[:3]):
        assert ref.off(a, b) <= tolerance(dtype)
    assert ref.off(back[4], want[4]) <= 2 * TOL
    room = 2 * TOL * float(want[3].norm() + (want[4] * exact[4].detach()).norm())
    assert float((back[3].cpu().double() - want[3]).norm()) <= room
    if float(want[5].norm()):
        assert ref.off(back[5], want[5]) <= TOL


@pytest.mark.parametrize("size", [SIZES[4], SIZES[7], SIZES[9]], ids=str)
def test_steps_give_what_the_rollout_gives(policy, size):
    x, state, starts = make(*size, seed=3)
    want_o, want_state = ref.rule(*x.values(), starts, state, size[4] ** -0.5)
    for t in range(size[1]):
        o = policy.gated_delta_step(*[a[:, t] for a in x.values()], state, starts=starts[:, t])
        assert ref.off(o, want_o[:, t]) <= tolerance(size[-1], 8 * TOL), t  # (a token's own norm is smaller)
    assert ref.off(state, want_state) <= TOL


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dims", [(64, 64), (128, 36), (100, 33), (31, 5)], ids=str)
def test_steps_of_views_at_any_address(policy, dims, dtype):
    """The same numbers in rows that 16-byte loads can read and in rows that they cannot."""
    x, state, starts = make(5, 2, 2, 4, *dims, dtype, seed=13)
    x = {n: t[:, 0].contiguous() for n, t in x.items()}
    whole = state.clone()
    want = policy.gated_delta_step(*x.values(), whole, starts=starts[:, 0])
    want_o, want_state = ref.rule(*[t[:, None] for t in x.values()], starts[:, :1], state, dims[0] ** -0.5)
    assert ref.off(want, want_o[:, 0]) <= tolerance(dtype)
    assert ref.off(whole, want_state) <= TOL
    for before, after in ((1, 0), (0, 3), (8, 8)):
        padded = {n: torch.nn.functional.pad(t, (before, after), value=math.nan) for n, t in x.items() if n in "qkv"}
        views = {n: padded[n][..., before:before + t.shape[-1]] if n in padded else t for n, t in x.items()}
        views["g"], views["beta"] = (x[n].t().contiguous().t() for n in ("g", "beta"))
        own = state.clone()
        assert torch.equal(policy.gated_delta_step(*views.values(), own, starts=starts[:, 0]), want)
        assert torch.equal(own, whole)


@pytest.mark.parametrize("kind", ["every token", "minus infinity", "decays of 1e4", "no writes", "all writes", "no decay",
                                  "one key"])
def test_extreme_gates(policy, kind):
    x, state, starts = make(2, 150, 1, 2, 64, 48, torch.float32, seed=5)
    starts = None
    if kind == "every token":
        starts = torch.ones(2, 150, dtype=torch.uint8, device="cuda")
    elif kind == "minus infinity":
        x["g"][:, ::37] = -math.inf
    elif kind == "decays of 1e4":
        x["g"][:, ::11] = -1e4
    elif kind == "no writes":
        x["beta"].zero_()
    elif kind == "all writes":
        x["beta"].fill_(1.0)
    elif kind == "no decay":
        x["g"].zero_()
    else:
        x["k"][:] = x["k"][:, :1]
    leaves = {n: t.clone().requires_grad_() for n, t in x.items()}
    s0 = state.clone().requires_grad_()
    o, final = policy.gated_delta_rule(*leaves.values(), starts=starts, initial_state=s0, return_state=True)
    exact = {n: t.detach().cpu().double().requires_grad_() for n, t in leaves.items()}
    e0 = s0.detach().cpu().double().requires_grad_()
    want_o, want_final = ref.rule(*exact.values(), starts, e0, 64 ** -0.5)
    assert ref.off(o, want_o) <= TOL
    assert ref.off(final, want_final) <= TOL
    go, gs = torch.randn_like(o), torch.randn_like(final)
    back = torch.autograd.grad([o, final], list(leaves.values()) + [s0], [go, gs])
    want = torch.autograd.grad([want_o, want_final], list(exact.values()) + [e0], [go.cpu().double(), gs.cpu().double()])
    scale = float((want[4] * exact["beta"].detach()).norm())
    for n, a, b in zip(list(leaves) + ["state"], back, want):
        b = torch.nan_to_num(b, nan=0.0) if n == "g" else b  # (exp(-inf) of autograd)
        assert torch.isfinite(a).all(), n
        room = 2 * TOL * (float(b.norm()) + (scale if n == "g" else 0.0)) + 1e-30
        assert float((a.cpu().double() - b).norm()) <= room, n


def test_a_start_forgets_a_state_that_is_not_finite(policy):
    x, state, _ = make(2, 100, 1, 1, 64, 64, torch.bfloat16)
    clean = state.clone()
    state[1] = math.nan
    state[1, :, 3] = math.inf
    starts = torch.zeros(2, 100, dtype=torch.bool, device="cuda")
    starts[1, 0] = True
    leaves = {n: t.clone().requires_grad_() for n, t in x.items()}
    o, final = policy.gated_delta_rule(*leaves.values(), starts=starts, initial_state=state, return_state=True)
    want, want_final = policy.gated_delta_rule(*x.values(), starts=starts, initial_state=clean, return_state=True)
    assert torch.equal(o, want) and torch.equal(final, want_final)
    back = torch.autograd.grad([o, final], list(leaves.values()), [torch.ones_like(o), torch.ones_like(final)])
    assert all(torch.isfinite(b).all() for b in back)
    stepped = policy.gated_delta_step(*[t[:, 0] for t in x.values()], state, starts=starts[:, 0])
    assert torch.isfinite(stepped).all() and torch.isfinite(state).all()


def test_views_of_one_projection_and_broadcasts(policy):
    size = (2, 130, 2, 2, 64, 32, torch.bfloat16)
    x, state, starts = make(*size, seed=7)
    packed = torch.cat([x["q"].flatten(2), x["k"].flatten(2), x["v"].flatten(2)], -1)
    odd = torch.empty(packed.numel() + 1, dtype=packed.dtype, device="cuda")[1:].view_as(packed).copy_(packed)
    for source in (packed, odd):  # 16-byte rows, and rows at odd addresses
        q, k, v = source.split([128, 128, 64], -1)
        q, k, v = q.unflatten(-1, (2, 64)), k.unflatten(-1, (2, 64)), v.unflatten(-1, (2, 32))
        wide = starts.clone()[:, :, None].expand(2, 130, 4)[:, :, 1]
        views = [t.detach().requires_grad_() for t in (q, k, v, x["g"].transpose(0, 1).contiguous().transpose(0, 1), x["beta"])]
        o = policy.gated_delta_rule(*views, starts=wide, initial_state=state)
        whole = [t.clone().requires_grad_() for t in x.values()]
        want = policy.gated_delta_rule(*whole, starts=starts, initial_state=state)
        assert torch.equal(o, want)
        got = torch.autograd.grad(o.float().sum(), views)  # a gradient of strides zero
        for a, b in zip(got, torch.autograd.grad(want, whole, torch.ones_like(want))):
            assert torch.equal(a, b)
    heads_first = x["v"].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(policy.gated_delta_rule(x["q"], x["k"], heads_first, x["g"], x["beta"]),
                       policy.gated_delta_rule(*x.values()))


def test_one_gate_for_all_heads(policy):
    x, _, _ = make(2, 70, 1, 4, 32, 32, torch.float32)
    g = x["g"][:, :, :1]
    gate = g.clone().requires_grad_()
    o = policy.gated_delta_rule(x["q"], x["k"], x["v"], gate.expand(2, 70, 4), x["beta"])
    assert torch.equal(o, policy.gated_delta_rule(x["q"], x["k"], x["v"], g.expand(2, 70, 4).contiguous(), x["beta"]))
    o.square().sum().backward()
    assert gate.grad.shape == gate.shape and torch.isfinite(gate.grad).all()


def test_one_query_and_one_value_for_all_steps(policy):
    """Expanded axes of steps, in a rollout that does not fill its last chunk."""
    x, state, _ = make(2, 70, 1, 1, 64, 64, torch.bfloat16)
    x = {n: t[:, :1].expand(t.shape) if n in "qv" else t for n, t in x.items()}
    leaves = [t.detach().requires_grad_() for t in x.values()]
    s0 = state.clone().requires_grad_()
    o = policy.gated_delta_rule(*leaves, initial_state=s0)
    whole = [t.contiguous().requires_grad_() for t in x.values()]
    s1 = state.clone().requires_grad_()
    want = policy.gated_delta_rule(*whole, initial_state=s1)
    assert torch.equal(o, want)
    for a, b in zip(torch.autograd.grad(o.float().sum(), leaves + [s0]),
                    torch.autograd.grad(want, whole + [s1], torch.ones_like(want))):
        assert torch.equal(a, b)


def test_far_offsets(policy):
    """Environments that lie more than 2^32 bytes apart."""
    x, _, starts = make(2, 66, 1, 1, 64, 64, torch.bfloat16)
    far = (1 << 31) + 64
    big = torch.empty(far + 66 * 192, dtype=torch.bfloat16, device="cuda")
    q, k, v = (big.as_strided((2, 66, 1, 64), (far, 192, 64, 1), 64 * i) for i in range(3))
    for t, n in zip((q, k, v), "qkv"):
        t.copy_(x[n])
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = policy.gated_delta_rule(*leaves, x["g"], x["beta"], starts=starts)
    whole = [x[n].clone().requires_grad_() for n in "qkv"]
    want = policy.gated_delta_rule(*whole, x["g"], x["beta"], starts=starts)
    assert torch.equal(o, want)
    for a, b in zip(torch.autograd.grad(o.float().square().sum(), leaves), torch.autograd.grad(want.float().square().sum(), whole)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("name", ["q", "k", "v", "g", "beta", "state"])
def test_gradients_against_differences(policy, name):
    """The loss along a direction: its slope by central differences of the kernel's own outputs.
    A step of 2^-6 leaves a cubic term of about 2^-12 of the slope and a rounding of the loss
    (of norm 1 per unit) of 2^-24 / 2^-6: within 1 part in 256 together."""
    x, state, starts = make(2, 90, 1, 2, 32, 32, torch.float32, seed=11)
    x["state"] = state
    gen = torch.Generator(device="cuda").manual_seed(1)
    weight = torch.randn(x["v"].shape, generator=gen, device="cuda")
    weight_state = torch.randn(state.shape, generator=gen, device="cuda")

    def loss(inputs):
        rest = {n: t for n, t in inputs.items() if n != "state"}
        o, final = policy.gated_delta_rule(*rest.values(), starts=starts, initial_state=inputs["state"], return_state=True)
        return (o.double() * weight).sum() + (final.double() * weight_state).sum()

    leaf = x[name].clone().requires_grad_()
    slope = torch.autograd.grad(loss({**x, name: leaf}), leaf)[0]
    direction = slope / slope.norm()
    h = 2.0 ** -6
    numeric = float(loss({**x, name: x[name] + h * direction}) - loss({**x, name: x[name] - h * direction})) / (2 * h)
    assert abs(numeric - float(slope.norm())) <= float(slope.norm()) / 256


def test_same_inputs_give_the_same_bits(policy):
    x, state, starts = make(3, 200, 2, 4, 64, 64, torch.bfloat16)

    def once():
        leaves = [t.clone().requires_grad_() for t in x.values()]
        o, final = policy.gated_delta_rule(*leaves, starts=starts, initial_state=state, return_state=True)
        return [o, final, *torch.autograd.grad([o, final], leaves, [torch.ones_like(o), torch.ones_like(final)])]

    first = once()
    for a, b in zip(first, once()):
        assert torch.equal(a, b)


def test_empty_batches_and_rollouts(policy):
    for envs, steps in ((0, 5), (2, 0)):
        x, state, starts = make(max(envs, 1), max(steps, 1), 1, 2, 16, 16, torch.float32)
        x = {n: t[:envs, :steps].contiguous() for n, t in x.items()}
        leaves = [t.requires_grad_() for t in x.values()]
        s0 = state[:envs].clone().requires_grad_()
        o, final = policy.gated_delta_rule(*leaves, starts=starts[:envs, :steps], initial_state=s0, return_state=True)
        assert o.shape == (envs, steps, 2, 16)
        assert torch.equal(final, s0)
        grads = torch.autograd.grad([o, final], leaves + [s0], [torch.ones_like(o), torch.ones_like(final)])
        assert torch.equal(grads[-1], torch.ones_like(s0))


def test_a_stream_of_its_own(policy):
    x, state, starts = make(4, 130, 1, 1, 64, 64, torch.bfloat16)
    want = policy.gated_delta_rule(*x.values(), starts=starts, initial_state=state)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [policy.gated_delta_rule(*x.values(), starts=starts, initial_state=state) for _ in range(8)]
    side.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_captured_steps_replay(policy):
    x, state, starts = make(4, 6, 1, 1, 64, 64, torch.bfloat16)
    start_state = state.clone()
    frame = {n: t[:, 0].clone() for n, t in x.items()}
    out = torch.empty_like(frame["v"])
    want = [policy.gated_delta_step(*[t[:, i] for t in x.values()], state).clone() for i in range(6)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        policy.gated_delta_step(*frame.values(), state, out=out)
    state.copy_(start_state)
    for i in range(6):
        for n in frame:
            frame[n].copy_(x[n][:, i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])


def test_captured_rollouts_replay(policy):
    x, state, starts = make(1, 64 * 17, 1, 2, 64, 64, torch.bfloat16)
    policy.gated_delta_rule(*x.values(), starts=starts, initial_state=state, return_state=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, final = policy.gated_delta_rule(*x.values(), starts=starts, initial_state=state, return_state=True)
    for n in range(4):
        x["v"].copy_(torch.randn(x["v"].shape, device="cuda"))
        state.normal_()
        want, want_final = policy.gated_delta_rule(*x.values(), starts=starts, initial_state=state, return_state=True)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.equal(final, want_final), n


def test_refusals(policy):
    x, state, starts = make(2, 8, 2, 4, 32, 32, torch.bfloat16)
    call = lambda **over: policy.gated_delta_rule(  # noqa: E731
        *[over.get(n, x[n]) for n in x], starts=over.get("starts", starts), initial_state=over.get("state", state))
    bad = [
        ({"q": x["q"].cpu()}, "q must be a CUDA tensor"),
        ({"q": x["q"].double()}, "q must be float32 or bfloat16 or float16"),
        ({"k": x["k"].float()}, "k must be bfloat16"),
        ({"v": x["v"].float()}, "v must be bfloat16"),
        ({"g": x["g"].half()}, "g must be float32"),
        ({"beta": x["beta"][:, :, :2]}, "beta must be"),
        ({"k": x["k"][:, :, :1]}, "q and k must both be"),
        ({"v": x["v"][:, :, :3]}, "multiple of the key heads"),
        ({"v": x["v"][:, :4]}, "v must be"),
        ({"q": x["q"].transpose(2, 3).contiguous().transpose(2, 3)}, "contiguous in its last dimension"),
        ({"starts": starts.int()}, "starts must be bool or uint8"),
        ({"starts": starts[:, :3]}, "starts must be"),
        ({"state": state.half()}, "initial_state must be float32"),
        ({"state": state[:1]}, "initial_state must be"),
        ({"state": state.transpose(2, 3)}, "initial_state must be contiguous"),
    ]
    for over, words in bad:
        with pytest.raises(RuntimeError, match=words):
            call(**over)
    wide = torch.zeros(2, 8, 2, 129, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="key dimension must be in"):
        call(q=wide, k=wide)
    frame = [t[:, 0] for t in x.values()]
    with pytest.raises(RuntimeError, match="no gradients"):
        policy.gated_delta_step(frame[0].clone().requires_grad_(), *frame[1:], state)
    with pytest.raises(RuntimeError, match="out must be"):
        policy.gated_delta_step(*frame, state, out=torch.empty(2, 4, 16, dtype=torch.bfloat16, device="cuda"))

"""The selective state space scan (``navi_amd.policy``) on the GPU against the recurrence in float64.

Tolerances. Products run on exact splits of float32 and accumulate in float32, so an output is a sum of
some hundred terms with relative errors of a few 2^-24 each: 32 x 2^-24 of the output's norm for
float32 values, and the output's own rounding on top where it is of 16 bits. The gradient of dt is
that of beta, a sum of the value's part and the decay's: 64 x 2^-24 of both. Gradients of a, d and
dt_bias are sums over tokens, whose terms have errors of either sign: 64 x 2^-24 of the terms'
absolute sum.
"""

from __future__ import annotations

import pytest
import torch

from . import block_reference as ref
from .policy_reference import EPS, off

pytestmark = pytest.mark.gpu

TOL = 32 * EPS
NAMES = ("x", "dt", "a", "b", "c", "d", "dt_bias")


@pytest.fixture(scope="module")
def policy(gpu):
    from navi_amd import policy

    return policy


def make(envs, steps, heads, groups, state_dim, head_dim, dtype, seed=0, often=0.04):
    gen = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    x = {"x": rand(envs, steps, heads, head_dim).to(dtype), "dt": 0.8 * rand(envs, steps, heads) - 3.0,
         "a": -torch.exp(1.5 * torch.rand(heads, generator=gen)), "b": rand(envs, steps, groups, state_dim).to(dtype),
         "c": rand(envs, steps, groups, state_dim).to(dtype), "d": 1.0 + rand(heads), "dt_bias": 0.5 * rand(heads)}
    state = 0.3 * rand(envs, heads, state_dim, head_dim)
    starts = torch.rand(envs, steps, generator=gen) < often
    return {k: v.cuda() for k, v in x.items()}, state.cuda(), starts.cuda()


def tolerance(t, base=TOL):
    return base + ref.rounding(t)


def call(policy, x, **rest):
    return policy.selective_scan(*[x[n] for n in ("x", "dt", "a", "b", "c")], d=x.get("d"), dt_bias=x.get("dt_bias"), **rest)


def reference(x, starts, state):
    return ref.scan(*[x[n] for n in ("x", "dt", "a", "b", "c")], x.get("d"), x.get("dt_bias"), starts, state)


def compare(policy, size, x, state, starts):
    """Outputs and gradients of all inputs."""
    dtype = size[-1]
    leaves = {n: t.clone().requires_grad_() for n, t in x.items()}
    s0 = None if state is None else state.clone().requires_grad_()
    got = call(policy, leaves, starts=starts, initial_state=s0, return_state=state is not None)
    y, final = got if state is not None else (got, None)
    exact = {n: t.detach().cpu().double() for n, t in leaves.items()}
    exact["a"] = exact["a"].expand(x["dt"].shape).clone()  # a rate for each token: what the gradient sums
    exact = {n: t.requires_grad_() for n, t in exact.items()}
    e0 = None if state is None else state.cpu().double().requires_grad_()
    want_y, want_final = reference(exact, starts, e0)
    assert y.dtype == dtype and off(y, want_y) <= tolerance(y)
    gen = torch.Generator().manual_seed(9)
    grads, outs, wants = [torch.randn(y.shape, generator=gen).to(dtype)], [y], [want_y]
    if state is not None:
        assert off(final, want_final) <= TOL
        grads.append(torch.randn(final.shape, generator=gen))
        outs.append(final)
        wants.append(want_final)
    given, exacts = [*leaves.values()], [*exact.values()]
    names = [*leaves]
    if state is not None:
        given, exacts, names = given + [s0], exacts + [e0], names + ["state"]
    back = dict(zip(names, torch.autograd.grad(outs, given, [t.cuda() for t in grads])))
    want = dict(zip(names, torch.autograd.grad(wants, exacts, [t.double() for t in grads])))
    for n in ("x", "b", "c"):
        assert back[n].dtype == dtype
        assert off(back[n], want[n]) <= tolerance(back[n]), n
    if state is not None:
        assert off(back["state"], want["state"]) <= TOL
    z = exact["dt"].detach() + exact.get("dt_bias", torch.zeros(())).detach()
    slope = torch.sigmoid(z) / (torch.clamp(z, min=0) + torch.log1p(torch.exp(-z.abs())))  # of log beta
    decay = (want["a"] * exact["a"].detach() * slope).abs()  # the decay's part of each token's gradient
    room = want["dt"].abs() + decay
    assert float((back["dt"].cpu().double() - want["dt"]).norm()) <= 2 * TOL * float(room.norm())
    terms = {"a": want["a"].abs().sum((0, 1)), "dt_bias": room.sum((0, 1)),
             "d": (grads[0].double().abs() * exact["x"].detach().abs()).sum((0, 1, 3))}
    for n, size_of in terms.items():
        if n in back:
            exact_sum = want["a"].sum((0, 1)) if n == "a" else want[n]
            assert ((back[n].cpu().double() - exact_sum).abs() <= 2 * TOL * size_of).all(), n
    return back


SIZES = [  # envs, steps, heads, groups, state_dim, head_dim
    (1, 1, 1, 1, 1, 1, torch.float32),
    (2, 1, 4, 2, 64, 64, torch.bfloat16),
    (3, 15, 2, 1, 16, 16, torch.float32),
    (2, 63, 2, 2, 64, 64, torch.float16),
    (2, 64, 1, 1, 64, 64, torch.float32),
    (1, 65, 3, 1, 33, 17, torch.float32),
    (2, 128, 2, 2, 64, 128, torch.bfloat16),
    (1, 129, 4, 2, 100, 72, torch.float16),
    (1, 130, 1, 1, 128, 128, torch.float32),
    (1, 257, 2, 1, 128, 64, torch.bfloat16),
    (5, 70, 3, 3, 7, 5, torch.bfloat16),
    (9, 192, 6, 3, 48, 80, torch.bfloat16),
]


@pytest.mark.parametrize("with_state", [False, True])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_scan_and_gradients(policy, size, with_state):
    x, state, starts = make(*size)
    back = compare(policy, size, x, state if with_state else None, starts if with_state else None)
    if with_state:  # (the decay of a token that begins an episode does nothing)
        assert torch.isfinite(back["dt"]).all()


@pytest.mark.parametrize("left_out", [("d",), ("dt_bias",), ("d", "dt_bias")])
def test_without_skip_or_bias(policy, left_out):
    size = (2, 90, 4, 2, 32, 48, torch.float32)
    x, state, starts = make(*size, seed=4)
    compare(policy, size, {n: t for n, t in x.items() if n not in left_out}, state, starts)


LONG = [  # few heads and many chunks: walked in segments that are joined
    (1, 64 * 8, 1, 1, 64, 64, torch.float32),
    (1, 64 * 9 + 5, 2, 1, 33, 70, torch.bfloat16),
    (2, 64 * 12 + 1, 2, 1, 128, 128, torch.float16),
    (9, 64 * 20 + 63, 2, 2, 20, 24, torch.bfloat16),
]


@pytest.mark.parametrize("ends", [True, False], ids=["episodes", "one episode"])
@pytest.mark.parametrize("size", LONG, ids=str)
def test_long_walks(policy, size, ends):
    x, state, starts = make(*size, seed=21, often=0.003)
    x["dt"] -= 3.0  # (a state that lasts through segments)
    compare(policy, size, x, state, starts if ends else None)


@pytest.mark.parametrize("steps", [1, 2, 4, 5])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_short_rollouts_without_gradients(policy, steps, dtype):
    x, state, starts = make(3, 6, 4, 2, 50, 36, dtype, seed=steps, often=0.3)
    x = {n: t[:, 1:1 + steps] if t.dim() > 1 else t for n, t in x.items()}  # (views)
    x["c"] = x["c"][:, :1].expand(x["c"].shape)
    starts = starts[:, 1:1 + steps]
    y, final = call(policy, x, starts=starts, initial_state=state, return_state=True)
    want_y, want_final = reference(x, starts, state)
    assert off(y, want_y) <= tolerance(y)
    assert off(final, want_final) <= TOL
    assert off(call(policy, x), reference(x, None, None)[0]) <= tolerance(y)


@pytest.mark.parametrize("size", [(1, 1, 1, 1, 1, torch.float32), (3, 4, 2, 50, 36, torch.bfloat16),
                                  (70, 6, 3, 33, 17, torch.float16), (2, 2, 1, 128, 128, torch.float32),
                                  (600, 8, 2, 64, 64, torch.bfloat16)], ids=str)
@pytest.mark.parametrize("given", [False, True], ids=["new", "out"])
def test_step(policy, size, given):
    envs, heads, groups, state_dim, head_dim, dtype = size
    x, state, starts = make(envs, 3, heads, groups, state_dim, head_dim, dtype, seed=5, often=0.3)
    want_y, want_final = reference(x, starts, state)
    carried, ys = state.clone(), []
    for t in range(3):
        args = [x["x"][:, t], x["dt"][:, t], x["a"], x["b"][:, t], x["c"][:, t], carried]
        if given:
            args[0] = args[0].contiguous()
        out = args[0] if given else None  # (x itself)
        got = policy.selective_scan_step(*args, d=x["d"], dt_bias=x["dt_bias"], starts=starts[:, t].to(torch.uint8), out=out)
        assert out is None or got is out
        ys.append(got)
    assert off(torch.stack(ys, 1), want_y) <= tolerance(torch.stack(ys, 1))
    assert off(carried, want_final) <= TOL


def test_views_of_one_projection_and_heads_before_steps(policy):
    gen = torch.Generator(device="cuda").manual_seed(2)
    for dtype in (torch.bfloat16, torch.float32):
        x, state, starts = make(2, 100, 4, 2, 32, 48, dtype, seed=6)
        whole = torch.randn(2, 100, 7 + 4 * 48 + 4 * 32, device="cuda", generator=gen).to(dtype)  # (rows at any address)
        x["x"] = whole[..., 7:7 + 192].unflatten(-1, (4, 48))
        x["b"], x["c"] = (whole[..., 199 + 64 * i:263 + 64 * i].unflatten(-1, (2, 32)) for i in range(2))
        x["dt"] = x["dt"].transpose(1, 2).contiguous().transpose(1, 2)
        strided = compare(policy, (2, 100, 4, 2, 32, 48, dtype), x, state, starts)
        dense = compare(policy, (2, 100, 4, 2, 32, 48, dtype), {n: t.contiguous() for n, t in x.items()}, state, starts)
        turned = {n: t.transpose(1, 2).contiguous().transpose(1, 2) if t.dim() == 4 else t for n, t in x.items()}
        other = compare(policy, (2, 100, 4, 2, 32, 48, dtype), turned, state, starts)
        for n in strided:
            assert torch.equal(strided[n], dense[n]) and torch.equal(strided[n], other[n]), n


def test_a_start_forgets_whatever_the_state_holds(policy):
    x, state, _ = make(2, 70, 2, 1, 16, 24, torch.float32, seed=8)
    starts = torch.zeros(2, 70, dtype=torch.bool, device="cuda")
    starts[:, 0] = True
    state.fill_(float("nan"))
    y, final = call(policy, x, starts=starts, initial_state=state, return_state=True)
    want_y, want_final = reference(x, None, None)
    assert off(y, want_y) <= TOL and off(final, want_final) <= TOL
    one = policy.selective_scan_step(x["x"][:, 0], x["dt"][:, 0], x["a"], x["b"][:, 0], x["c"][:, 0], state, d=x["d"],
                                     dt_bias=x["dt_bias"], starts=starts[:, 0])
    assert off(one, want_y[:, 0]) <= TOL and torch.isfinite(state).all()


def test_rates_without_end_clear_the_state(policy):
    x, state, _ = make(2, 130, 3, 1, 16, 24, torch.float32, seed=9)
    x["a"] = torch.tensor([-float("inf"), -3.0, -1e30], device="cuda")
    y, final = call(policy, x, initial_state=state, return_state=True)
    want_y, want_final = reference(x, None, state)
    assert off(y, want_y) <= TOL and off(final, want_final) <= TOL


def test_empty(policy):
    x, state, starts = make(2, 3, 4, 2, 8, 6, torch.bfloat16)
    none = {n: t[:, :0] if t.dim() > 1 else t for n, t in x.items()}
    leaves = {n: t.clone().requires_grad_() for n, t in none.items()}
    s0 = state.clone().requires_grad_()
    y, final = call(policy, leaves, initial_state=s0, return_state=True)
    assert y.shape == (2, 0, 4, 6) and torch.equal(final, state)
    grads = torch.autograd.grad([y, final], [*leaves.values(), s0], [y.detach(), torch.ones_like(final)])
    assert torch.equal(grads[-1], torch.ones_like(state)) and not grads[2].any() and not grads[5].any()
    nobody = {n: t[:0] if t.dim() > 1 else t for n, t in x.items()}
    y, final = call(policy, nobody, return_state=True)
    assert y.shape == (0, 3, 4, 6) and final.shape == (0, 4, 8, 6)
    policy.selective_scan_step(*[nobody[n][:, 0] if nobody[n].dim() > 1 else nobody[n] for n in ("x", "dt", "a", "b", "c")], final)


def test_gradients_of_some_inputs_are_the_same_numbers(policy):
    x, state, starts = make(3, 200, 4, 2, 24, 40, torch.bfloat16, seed=11)
    every = {**x, "state": state}

    def run(wanted):
        leaves = {n: t.clone().requires_grad_(n in wanted) for n, t in every.items()}
        s0 = leaves.pop("state")
        y, final = call(policy, leaves, starts=starts, initial_state=s0, return_state=True)
        leaves["state"] = s0
        gen = torch.Generator(device="cuda").manual_seed(1)
        grads = [torch.randn(t.shape, device="cuda", generator=gen).to(t.dtype) for t in (y, final)]
        return dict(zip(wanted, torch.autograd.grad([y, final], [leaves[n] for n in wanted], grads)))

    want = run([*every])
    for wanted in (["x"], ["dt", "a"], ["state"], ["dt_bias"], ["b", "d"]):
        for n, g in run(wanted).items():
            assert torch.equal(g, want[n]), n


def test_gradients_of_one_output(policy):
    x, state, starts = make(2, 150, 2, 1, 24, 40, torch.float32, seed=12)
    for which in (0, 1):
        leaves = {n: t.clone().requires_grad_() for n, t in x.items()}
        exact = {n: t.cpu().double().requires_grad_() for n, t in x.items()}
        out = call(policy, leaves, starts=starts, initial_state=state, return_state=True)[which]
        want = reference(exact, starts, state)[which]
        g = torch.randn(out.shape, generator=torch.Generator().manual_seed(3))
        names = ["x", "b"]
        got = torch.autograd.grad(out, [leaves[n] for n in names], g.cuda())
        for a, b in zip(got, torch.autograd.grad(want, [exact[n] for n in names], g.double())):
            assert off(a, b) <= TOL


def test_gradients_against_differences(policy):
    """Along a random direction: the difference of second order at distance h leaves about h^2 / 6 of
    the third derivative (of size 1 beside the first here), float32 sums of 2^13 numbers 2^-24 sqrt(2^13) / h of
    the outputs' norm: with h = 2^-7, 2^-17 and 2^-11 of numbers of the derivative's size or a few times it."""
    x, state, starts = make(2, 100, 2, 1, 16, 20, torch.float32, seed=13)
    gen = torch.Generator(device="cuda").manual_seed(3)
    every = {**x, "state": state}
    way = {n: torch.randn(t.shape, device="cuda", generator=gen) for n, t in every.items()}
    weight = torch.randn(x["x"].shape, device="cuda", generator=gen)

    def loss(at):
        at = dict(at)
        s0 = at.pop("state")
        y, final = call(policy, at, starts=starts, initial_state=s0, return_state=True)
        return (y.double() * weight).sum() + final.double().sum()

    leaves = {n: t.clone().requires_grad_() for n, t in every.items()}
    grads = dict(zip(every, torch.autograd.grad(loss(leaves), [*leaves.values()])))
    h = 2.0 ** -7
    for n in every:
        there, back = ({**every, n: every[n] + s * h * way[n]} for s in (1, -1))
        difference = float(loss(there) - loss(back)) / (2 * h)
        slope = float((grads[n].double() * way[n]).sum())
        scale = float((grads[n].double() * way[n]).norm())
        assert abs(difference - slope) <= 2.0 ** -8 * max(scale, abs(slope)), n


def test_sixteen_bit_results_are_rounded_once(policy):
    """Of outputs and gradients before their rounding nothing coarser than 32 x 2^-24 is lost: no more
    numbers differ from the exact ones' rounding than lie so near to a border (2 x 32 x 2^-24 of 2^-8 or
    2^-11 apart, one in 2^10 or 2^7; twice that)."""
    for dtype, share in ((torch.bfloat16, 2.0 ** -9), (torch.float16, 2.0 ** -6)):
        x, state, starts = make(3, 200, 4, 2, 64, 64, dtype, seed=14)
        leaves = {n: t.clone().requires_grad_() for n, t in x.items()}
        y = call(policy, leaves, starts=starts, initial_state=state)
        exact = {n: t.cpu().double().requires_grad_() for n, t in x.items()}
        want = reference(exact, starts, state)[0]
        g = torch.randn(y.shape, generator=torch.Generator().manual_seed(3)).to(dtype)
        names = ["x", "b", "c"]
        pairs = [(y, want), *zip(torch.autograd.grad(y, [leaves[n] for n in names], g.cuda()),
                                 torch.autograd.grad(want, [exact[n] for n in names], g.double()))]
        for got, exactly in pairs:
            big = exactly.detach().abs() > 0.1 * exactly.detach().abs().mean()
            assert float((got.cpu() != exactly.detach().to(dtype))[big].double().mean()) <= share


def test_sums_over_many_tokens_have_no_bias(policy):
    """Gradients of a and dt_bias of 131072 tokens of either sign, to within what random errors of
    2^-22 of each token's gradient leave (four times their spread): matrix sums that lie to one side would show."""
    x, _, starts = make(512, 128, 2, 1, 32, 32, torch.bfloat16, seed=15)
    x["b"], x["c"], x["x"] = (torch.nn.functional.silu(x[n].float()).to(torch.bfloat16) for n in ("b", "c", "x"))
    leaves = {n: t.clone().requires_grad_() for n, t in x.items()}
    y = call(policy, leaves, starts=starts)
    exact = {n: t.detach().cpu().double() for n, t in leaves.items()}
    exact["a"] = exact["a"].expand(x["dt"].shape).clone()
    exact = {n: t.requires_grad_() for n, t in exact.items()}
    g = torch.randn(y.shape, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    got = dict(zip(("a", "dt_bias"), torch.autograd.grad(y, [leaves["a"], leaves["dt_bias"]], g.cuda())))
    want = torch.autograd.grad(reference(exact, starts, None)[0], [exact["a"], exact["dt"]], g.double())
    for n, each in zip(got, want):
        spread = each.square().sum((0, 1)).sqrt() + (want[1].square().sum((0, 1)).sqrt() if n == "dt_bias" else 0)
        assert ((got[n].cpu().double() - each.sum((0, 1))).abs() <= 4 * 2.0 ** -22 * spread + EPS * each.sum((0, 1)).abs()).all(), n

"""What stands between two blocks (``navi_amd.policy.block_norm``) on the GPU against its definition in float64.

Tolerances: each number comes from a few float32 operations and two sums over a row: 16 x 2^-24 of the
norm (the backward pass, with four sums, 32), and its own rounding where it is of 16 bits. The gradient
through a norm is r (f - n mean(f n)), a difference whose two parts may be far larger than it (a row of
one number has none but through eps), and so is silu's slope: there the parts' norm counts as well. Gradients of the
vectors are sums over rows, 32 x 2^-24 of the terms' absolute sum for the terms and as much for the sums.
"""

from __future__ import annotations

import pytest
import torch

from . import block_reference as ref
from .policy_reference import EPS, off

pytestmark = pytest.mark.gpu

TOL = 16 * EPS
NAMES = ("y", "residual", "gate", "scale", "post_weight", "pre_weight")


@pytest.fixture(scope="module")
def policy(gpu):
    from navi_amd import policy

    return policy


def make(envs, steps, width, dtype, stream, seed=0):
    gen = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    rows = (envs, steps, width)
    x = {"y": rand(*rows).to(dtype), "residual": rand(*rows).to(stream), "gate": rand(*rows).to(dtype),
         "scale": 0.5 + 0.2 * rand(width), "post_weight": 1 + 0.2 * rand(width), "pre_weight": 1 + 0.2 * rand(width)}
    return {n: t.cuda() for n, t in x.items()}


def tolerance(t, base=TOL):
    return base + ref.rounding(t)


def compare(policy, x, eps=1e-6):
    leaves = {n: t.clone().requires_grad_() if t.is_contiguous() else t.detach().requires_grad_() for n, t in x.items()}
    exact = {n: t.detach().cpu().double().requires_grad_() for n, t in x.items()}
    rest = {n: leaves.get(n) for n in NAMES[2:]}
    got = policy.block_norm(leaves["y"], leaves["residual"], eps=eps, **rest)
    *want, first, second = ref.block(*[exact.get(n) for n in NAMES], eps, parts=True)
    dtype, stream = x["y"].dtype, x["residual"].dtype
    assert got[0].dtype == stream and got[1].dtype == dtype
    for g, w in zip(got, want):
        assert off(g, w) <= tolerance(g)
    gen = torch.Generator().manual_seed(9)
    grads = [torch.randn(g.shape, generator=gen).to(g.dtype) for g in got]
    back = dict(zip(leaves, torch.autograd.grad(got, [*leaves.values()], [g.cuda() for g in grads])))
    wanted = dict(zip(exact, torch.autograd.grad(want, [*exact.values()], [g.double() for g in grads], retain_graph=True)))
    through = torch.autograd.grad(want, [first, second], [g.double() for g in grads])
    inverse = [1 / torch.sqrt(t.detach().double().cpu().square().mean(-1, keepdim=True) + eps) for t in (x["y"], want[0])]
    parts = dict(zip(("y", "residual"), [f * r for f, r in zip(through, inverse)]))
    if "gate" in x:  # silu' = s + z s (1 - s), a difference for z below 0, times dh, one of those above
        z = exact["gate"].detach()
        along = first.detach() * (exact["scale"].detach() if "scale" in x else 1) * (exact["post_weight"].detach() if "post_weight" in x else 1)
        parts["gate"] = (wanted["residual"].abs() + parts["residual"].abs()) * along.abs() * torch.sigmoid(z) * (1 + z.abs())
    for n in ("y", "residual", "gate"):
        if n in x:
            room = tolerance(back[n], 2 * TOL) * wanted[n].norm() + (2 * TOL * parts[n].norm() if n in parts else 0.0)
            assert float((back[n].cpu().double() - wanted[n]).norm()) <= float(room), n
    # sums over rows of dh m, dh scale silu n and dnormed n: sizes of the terms, with those of dh's parts
    # (what a row's sums leave out is spread over the row)
    factor = lambda n: exact[n].detach() if n in x else torch.ones((), dtype=torch.float64)  # noqa: E731
    silu = exact["gate"].detach() * torch.sigmoid(exact["gate"].detach()) if "gate" in x else torch.ones((), dtype=torch.float64)
    dh = wanted["residual"].abs() + parts["residual"].abs()
    dh = dh + dh.mean(-1, keepdim=True)
    sizes = {"scale": dh * (first.detach() * factor("post_weight") * silu).abs(),
             "post_weight": dh * (first.detach() * factor("scale") * silu).abs(),
             "pre_weight": (grads[1].double() * second.detach()).abs()}
    for n, size in sizes.items():
        if n in x:
            assert ((back[n].cpu().double() - wanted[n]).abs() <= 64 * EPS * size.sum((0, 1))).all(), n
    return got, back


SIZES = [
    (1, 1, 1, torch.float32, torch.float32),
    (2, 3, 64, torch.bfloat16, torch.float32),
    (3, 5, 128, torch.float16, torch.float16),
    (7, 33, 256, torch.bfloat16, torch.bfloat16),
    (2, 9, 100, torch.float32, torch.float32),
    (5, 7, 512, torch.float32, torch.float32),
    (2, 20, 1000, torch.bfloat16, torch.float32),
    (3, 4, 777, torch.float16, torch.float32),
    (2, 5, 2048, torch.bfloat16, torch.bfloat16),
    (1, 3, 4095, torch.float32, torch.float32),
    (1, 2, 8192, torch.bfloat16, torch.float32),
    (40, 64, 192, torch.bfloat16, torch.float32),
]


@pytest.mark.parametrize("size", SIZES, ids=str)
def test_outputs_and_gradients(policy, size):
    compare(policy, make(*size))


@pytest.mark.parametrize("left_out", [("gate",), ("scale",), ("post_weight",), ("pre_weight",), NAMES[2:]], ids=str)
def test_parts_that_are_left_out(policy, left_out):
    x = make(3, 20, 192, torch.bfloat16, torch.float32, seed=2)
    compare(policy, {n: t for n, t in x.items() if n not in left_out})


def test_rows_of_zeros(policy):
    x = make(2, 4, 96, torch.float32, torch.float32, seed=3)
    x["y"][:, 1] = 0
    x["residual"][:, 1] = 0
    compare(policy, x, eps=1e-5)
    stream, normed = policy.block_norm(torch.zeros(1, 2, 64, device="cuda"), torch.zeros(1, 2, 64, device="cuda"), eps=1e-6)
    assert not stream.any() and not normed.any()


def test_strides_and_alignment_change_nothing(policy):
    for dtype in (torch.float32, torch.bfloat16):
        x = make(3, 20, 64, dtype, torch.float32, seed=4)
        want, back = compare(policy, x)
        for at in (0, 3, 8):
            there = {}
            for n, t in x.items():
                if t.dim() == 3:
                    wide = torch.zeros(3, 20, 80, dtype=t.dtype, device="cuda")
                    there[n] = wide[..., at:at + 64]
                    there[n].copy_(t)
                else:
                    there[n] = t
            got, other = compare(policy, there)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            assert all(torch.equal(other[n], back[n]) for n in ("y", "residual", "gate"))
        turned = {n: t.transpose(0, 1).contiguous().transpose(0, 1) if t.dim() == 3 else t for n, t in x.items()}
        got, _ = compare(policy, turned)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_gradients_of_one_output_and_of_some_inputs(policy):
    x = make(4, 30, 192, torch.bfloat16, torch.float32, seed=5)
    for which in (0, 1):
        leaves = {n: t.clone().requires_grad_() for n, t in x.items()}
        exact = {n: t.cpu().double().requires_grad_() for n, t in x.items()}
        got = policy.block_norm(leaves["y"], leaves["residual"], **{n: leaves[n] for n in NAMES[2:]})[which]
        want = ref.block(*[exact[n] for n in NAMES], 1e-6)[which]
        g = torch.randn(got.shape, generator=torch.Generator().manual_seed(1)).to(got.dtype)
        names = NAMES[:3]
        for n, a, b in zip(names, torch.autograd.grad(got, [leaves[n] for n in names], g.cuda(), retain_graph=True),
                           torch.autograd.grad(want, [exact[n] for n in names], g.double())):
            assert off(a, b) <= tolerance(a, 2 * TOL), n
        some = {n: t.clone().requires_grad_(n in ("gate", "scale")) for n, t in x.items()}
        again = policy.block_norm(some["y"], some["residual"], **{n: some[n] for n in NAMES[2:]})[which]
        every = torch.autograd.grad(got, [leaves["gate"], leaves["scale"]], g.cuda())
        for a, b in zip(torch.autograd.grad(again, [some["gate"], some["scale"]], g.cuda()), every):
            assert torch.equal(a, b)
    broadcast = policy.block_norm(leaves["y"], leaves["residual"])[0]
    (back,) = torch.autograd.grad(broadcast.sum(), leaves["residual"])  # (an expanded gradient)
    assert torch.equal(back, torch.ones_like(back))


def test_empty(policy):
    x = make(2, 3, 64, torch.bfloat16, torch.float32)
    for cut in (lambda t: t[:0], lambda t: t[:, :0]):
        leaves = {n: (cut(t) if t.dim() == 3 else t).clone().requires_grad_() for n, t in x.items()}
        stream, normed = policy.block_norm(leaves["y"], leaves["residual"], **{n: leaves[n] for n in NAMES[2:]})
        assert stream.shape == cut(x["y"]).shape == normed.shape
        grads = torch.autograd.grad([stream, normed], [*leaves.values()], [stream.detach(), normed.detach()])
        assert not any(g.any() for g in grads)


def test_gradients_against_differences(policy):
    """As for the convolution: 2^-8 of the slope's size at h = 2^-6."""
    x = make(2, 10, 40, torch.float32, torch.float32, seed=7)
    gen = torch.Generator(device="cuda").manual_seed(3)
    ways = {n: torch.randn(t.shape, device="cuda", generator=gen) for n, t in x.items()}
    weights = [torch.randn(x["y"].shape, device="cuda", generator=gen) for _ in range(2)]

    def loss(at):
        got = policy.block_norm(at["y"], at["residual"], **{n: at[n] for n in NAMES[2:]})
        return sum((g.double() * w).sum() for g, w in zip(got, weights))

    leaves = {n: t.clone().requires_grad_() for n, t in x.items()}
    grads = dict(zip(x, torch.autograd.grad(loss(leaves), [*leaves.values()])))
    h = 2.0 ** -6
    for n in x:
        there, back = ({**x, n: x[n] + s * h * ways[n]} for s in (1, -1))
        slope = grads[n].double() * ways[n]
        assert abs(float(loss(there) - loss(back)) / (2 * h) - float(slope.sum())) <= 2.0 ** -8 * max(float(slope.norm()), abs(float(slope.sum()))), n

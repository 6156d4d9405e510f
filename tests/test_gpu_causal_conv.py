"""The short convolution (``navi_amd.policy``) on the GPU against its definition in float64.

Tolerances: a number is a sum of up to five products in float32 and an activation of a few operations,
8 x 2^-24 of the norm, and its own rounding where it is of 16 bits; gradients of weight and bias are sums over
tokens, in float32 over a lane's tokens and a workgroup's rows: 32 x 2^-24 of the terms' absolute sum.
"""

from __future__ import annotations

import pytest
import torch

from . import block_reference as ref
from .policy_reference import EPS, off

pytestmark = pytest.mark.gpu

TOL = 8 * EPS


@pytest.fixture(scope="module")
def policy(gpu):
    from navi_amd import policy

    return policy


def make(envs, steps, channels, taps, dtype, seed=0, often=0.1):
    gen = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    x = rand(envs, steps, channels).to(dtype)
    return [t.cuda() for t in (x, rand(channels, taps), rand(channels), rand(envs, taps - 1, channels).to(dtype),
                               torch.rand(envs, steps, generator=gen) < often)]


def tolerance(t):
    return TOL + ref.rounding(t)


SIZES = [  # envs, steps, channels, taps
    (1, 1, 1, 2, torch.float32),
    (2, 2, 8, 4, torch.bfloat16),
    (3, 7, 20, 3, torch.float32),
    (2, 64, 33, 4, torch.float16),
    (2, 65, 64, 2, torch.bfloat16),
    (70, 130, 48, 4, torch.bfloat16),
    (1, 1000, 2056, 4, torch.float32),
    (5, 9, 4100, 3, torch.float16),
    (300, 3, 16, 4, torch.float32),
]


def compare(policy, x, weight, bias, window, starts, activation, dtype):
    given = [t for t in (x, weight, bias, window) if t is not None]
    leaves = [None if t is None else t.clone().requires_grad_() for t in (x, weight, bias, window)]
    exact = [None if t is None else t.cpu().double().requires_grad_() for t in (x, weight, bias, window)]
    y, after = policy.causal_conv(leaves[0], leaves[1], bias=leaves[2], starts=starts, initial_window=leaves[3], return_window=True,
                                  activation=activation)
    want_y, want_after = ref.conv(exact[0], exact[1], exact[2], starts, exact[3], activation)
    assert y.dtype == dtype and off(y, want_y) <= tolerance(y)
    assert torch.equal(after.cpu().double(), want_after.detach())
    gen = torch.Generator().manual_seed(9)
    grads = [torch.randn(t.shape, generator=gen).to(dtype) for t in (y, after)]
    back = torch.autograd.grad([y, after], [t for t in leaves if t is not None], [g.cuda() for g in grads])
    want = torch.autograd.grad([want_y, want_after], [t for t in exact if t is not None], [g.double() for g in grads])
    assert off(back[0], want[0]) <= tolerance(back[0])
    if window is not None:
        assert off(back[-1], want[-1]) <= tolerance(back[-1])
    # the terms of the sums: gradients of the same products with everything positive, 1.1 the activation's steepest slope
    size = [t.detach().abs().requires_grad_() for t in exact if t is not None]
    named = dict(zip([n for n, t in zip("xwbh", exact) if t is not None], size))
    total, _ = ref.conv(named["x"], named["w"], named.get("b"), starts, named.get("h"), None)
    room = torch.autograd.grad(total, [t for n, t in named.items() if n in "wb"], 1.1 * grads[0].double().abs())
    for got, exactly, most in zip(back[1:], want[1:], room):
        assert ((got.cpu().double() - exactly).abs() <= 32 * EPS * most).all()
    return y, after, back


@pytest.mark.parametrize("full", [True, False], ids=["everything", "weight alone"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_convolution_and_gradients(policy, size, full):
    x, weight, bias, window, starts = make(*size)
    if full:
        compare(policy, x, weight, bias, window, starts, "silu", size[-1])
    else:
        compare(policy, x, weight, None, None, None, None, size[-1])


@pytest.mark.parametrize("size", [(1, 1, 2, torch.float32), (3, 20, 3, torch.bfloat16), (64, 384, 4, torch.float16),
                                  (1030, 48, 4, torch.float32)], ids=str)
@pytest.mark.parametrize("given", [False, True], ids=["new", "out"])
def test_step(policy, size, given):
    envs, channels, taps, dtype = size
    x, weight, bias, window, starts = make(envs, 6, channels, taps, dtype, often=0.3)
    want_y, want_window = ref.conv(x, weight, bias, starts, window, "silu")
    ys = []
    for t in range(6):
        frame = x[:, t].contiguous() if given else x[:, t]
        out = frame if given else None  # (x itself)
        ys.append(policy.causal_conv_step(frame, weight, window, bias=bias, starts=starts[:, t], out=out))
        assert out is None or ys[-1] is out
    assert off(torch.stack(ys, 1), want_y) <= tolerance(torch.stack(ys, 1))
    assert torch.equal(window.cpu().double(), want_window)


def test_nothing_of_another_episode_is_read(policy):
    """Infinities and NaN before a start do not reach what follows."""
    for dtype in (torch.float32, torch.bfloat16):
        x, weight, bias, window, _ = make(2, 90, 16, 4, dtype)
        starts = torch.zeros(2, 90, dtype=torch.uint8, device="cuda")
        starts[:, 40] = 1
        spoiled, clean = x.clone(), x.clone()
        spoiled[:, 37:40] = torch.tensor([float("nan"), float("inf"), -float("inf")], device="cuda")[:, None]
        window = torch.full_like(window, float("nan"))
        got, after = policy.causal_conv(spoiled, weight, bias=bias, starts=starts, initial_window=window, return_window=True)
        want = policy.causal_conv(clean, weight, bias=bias, starts=starts)
        assert torch.equal(got[:, 40:], want[:, 40:]) and torch.isfinite(after).all()
        first = torch.zeros_like(starts)
        first[:, 0] = 1
        assert torch.isfinite(policy.causal_conv(clean, weight, bias=bias, starts=first, initial_window=window)).all()
        # gradients of inputs before the start: none of what follows, and theirs nothing of that
        leaf = clean.clone().requires_grad_()
        y = policy.causal_conv(leaf, weight, bias=bias, starts=starts)
        (back,) = torch.autograd.grad(y[:, 40:].float().sum(), leaf)
        assert not back[:, :40].any() and back[:, 40:].abs().sum() > 0


def test_strides_and_alignment_change_nothing(policy):
    for dtype in (torch.float32, torch.bfloat16):
        x, weight, bias, window, starts = make(3, 50, 64, 4, dtype, seed=4)
        want = compare(policy, x, weight, bias, window, starts, "silu", dtype)
        wide = torch.zeros(3, 50, 80, dtype=dtype, device="cuda")
        for at in (0, 5, 8):
            wide[..., at:at + 64] = x
            got = compare(policy, wide[..., at:at + 64], weight, bias, window, starts, "silu", dtype)
            assert torch.equal(got[0], want[0]) and all(torch.equal(a, b) for a, b in zip(got[2][:1], want[2][:1]))
        turned = x.transpose(0, 1).contiguous().transpose(0, 1)
        assert torch.equal(policy.causal_conv(turned, weight, bias=bias, starts=starts, initial_window=window), want[0])
        every = starts.t().contiguous().t()
        assert torch.equal(policy.causal_conv(x, weight, bias=bias, starts=every, initial_window=window), want[0])
        one = x[:, :1].expand(3, 50, 64)
        assert torch.equal(policy.causal_conv(one, weight), policy.causal_conv(one.contiguous(), weight))


def test_empty(policy):
    x, weight, bias, window, _ = make(2, 3, 8, 4, torch.bfloat16)
    leaf, held = x[:, :0].clone().requires_grad_(), window.clone().requires_grad_()
    w = weight.clone().requires_grad_()
    y, after = policy.causal_conv(leaf, w, bias=bias, initial_window=held, return_window=True)
    assert y.shape == (2, 0, 8) and torch.equal(after, window)
    grads = torch.autograd.grad([y, after], [leaf, w, held], [y.detach(), torch.ones_like(after)])
    assert not grads[1].any() and torch.equal(grads[2], torch.ones_like(window))
    assert not policy.causal_conv(x[:, :0], weight, return_window=True)[1].any()
    assert policy.causal_conv(x[:0], weight).shape == (0, 3, 8)


def test_gradients_against_differences(policy):
    """The difference of second order at h = 2^-6 leaves h^2 / 6 of the third derivative, float32's sums
    2^-24 / h: both below 2^-10 of the derivative's size; the directions' cancellation within 2^-8."""
    x, weight, bias, window, starts = make(2, 60, 12, 4, torch.float32, seed=7)
    gen = torch.Generator(device="cuda").manual_seed(3)
    at = [x, weight, bias, window]
    ways = [torch.randn(t.shape, device="cuda", generator=gen) for t in at]
    weights = torch.randn(x.shape, device="cuda", generator=gen)

    def loss(x, weight, bias, window):
        y, after = policy.causal_conv(x, weight, bias=bias, starts=starts, initial_window=window, return_window=True)
        return (y.double() * weights).sum() + after.double().sum()

    leaves = [t.clone().requires_grad_() for t in at]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    h = 2.0 ** -6
    for i, (g, way) in enumerate(zip(grads, ways)):
        there, back = ([t + s * h * way if i == j else t for j, t in enumerate(at)] for s in (1, -1))
        slope = (g.double() * way)
        assert abs(float(loss(*there) - loss(*back)) / (2 * h) - float(slope.sum())) <= 2.0 ** -8 * max(float(slope.norm()), abs(float(slope.sum())))

"""The convolution and the block norms at the ends of their ranges, against float64."""

from __future__ import annotations

import pytest
import torch

from . import block_reference as ref
from .policy_reference import EPS, off

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def policy(gpu):
    from navi_amd import policy

    return policy


@pytest.mark.parametrize("channels", [65536, 65535])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_as_many_channels_as_there_may_be(policy, channels, dtype):
    """Outputs are sums of five terms with a few 2^-24 each, gradients of the weights sums over 22 tokens."""
    gen = torch.Generator().manual_seed(1)
    rand = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    x, window, grad = rand(2, 11, channels).to(dtype), rand(2, 3, channels).to(dtype), rand(2, 11, channels).to(dtype)
    weight, bias, starts = 0.5 * rand(channels, 4), rand(channels), torch.rand(2, 11, generator=gen) < 0.1
    leaves = [t.cuda().requires_grad_() for t in (x, weight, bias, window)]
    y = policy.causal_conv(leaves[0], leaves[1], bias=leaves[2], starts=starts.cuda(), initial_window=leaves[3])
    exact = [t.double().requires_grad_() for t in (x, weight, bias, window)]
    want, _ = ref.conv(exact[0], exact[1], exact[2], starts, exact[3], "silu")
    assert off(y, want) <= 32 * EPS + ref.rounding(y)
    for got, exactly in zip(torch.autograd.grad(y, leaves, grad.cuda()), torch.autograd.grad(want, exact, grad.double())):
        assert off(got, exactly) <= 32 * EPS + ref.rounding(got)
    frame = window.cuda()
    got = policy.causal_conv_step(x[:, 0].cuda(), weight.cuda(), frame, bias=bias.cuda(), starts=starts[:, 0].cuda())
    assert off(got, want[:, 0]) <= 32 * EPS + ref.rounding(got)


def test_more_workgroups_than_a_launch_has(policy):
    """A frame of more environments than 2^24 workgroups of one row each hold: some take several."""
    gen = torch.Generator().manual_seed(3)
    envs = (1 << 23) + 5
    x, weight = torch.randn(3, 1, 257, generator=gen).to(torch.bfloat16), torch.randn(257, 2, generator=gen)
    rows = torch.zeros(envs, dtype=torch.long, device="cuda")
    rows[[1, 77, 1 << 20, envs - 6, envs - 1]] = 1
    rows[[3, 1 << 22, envs - 7, envs - 2]] = 2
    y = policy.causal_conv(x.cuda()[rows], weight.cuda())
    want = ref.conv(x, weight, None, None, None, "silu")[0]
    assert off(y[rows.nonzero().flatten()], want[rows[rows.nonzero().flatten()].cpu()]) <= 32 * EPS + ref.rounding(y)
    assert off(y[0], want[0]) <= 32 * EPS + 2.0 ** -8
    assert torch.equal(y.flatten(1).view(torch.int16).sum(1)[rows == 0].unique(), y[0].view(torch.int16).sum().flatten())


@pytest.mark.parametrize("width", [8192, 8191])
def test_rows_as_wide_as_there_may_be(policy, width):
    gen = torch.Generator().manual_seed(2)
    rand = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    given = [rand(2, 3, width), rand(2, 3, width), rand(2, 3, width), rand(width), rand(width), rand(width)]
    leaves = [t.cuda().requires_grad_() for t in given]
    got = policy.block_norm(leaves[0], leaves[1], gate=leaves[2], scale=leaves[3], post_weight=leaves[4], pre_weight=leaves[5])
    exact = [t.double().requires_grad_() for t in given]
    want = ref.block(*exact, 1e-6)
    grads = [rand(2, 3, width), rand(2, 3, width)]
    for a, b in zip(got, want):
        assert off(a, b) <= 32 * EPS
    for a, b in zip(torch.autograd.grad(got, leaves, [t.cuda() for t in grads]), torch.autograd.grad(want, exact, [t.double() for t in grads])):
        assert off(a, b) <= 64 * EPS

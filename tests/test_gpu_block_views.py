"""Views of the convolution's inputs whose steps lie far apart."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def policy(gpu):
    from navi_amd import policy

    return policy


def far(t, gen_seed):
    """The same numbers (of 16 bits) in a rollout whose steps are 64 MiB apart, 2.5 GiB from the first to the last."""
    envs, steps, channels = t.shape
    store = torch.empty(steps << 25, dtype=t.dtype, device="cuda")
    view = store.as_strided((envs, steps, channels), (channels + 8 * gen_seed, 1 << 25, 1))
    return view.copy_(t)


def test_a_convolution_over_steps_far_apart(policy):
    gen = torch.Generator().manual_seed(0)
    x, grad = (torch.randn(3, 41, 16, generator=gen).to(torch.bfloat16).cuda() for _ in range(2))
    weight, starts = torch.randn(16, 4, generator=gen).cuda(), (torch.rand(3, 41, generator=gen) < 0.1).cuda()
    want_leaf, weight_leaf = x.clone().requires_grad_(), weight.clone().requires_grad_()
    want = policy.causal_conv(want_leaf, weight_leaf, starts=starts)
    want_grads = torch.autograd.grad(want, [want_leaf, weight_leaf], grad)
    leaf, weight_again = far(x, 0).requires_grad_(), weight.clone().requires_grad_()
    got = policy.causal_conv(leaf, weight_again, starts=starts)
    grads = torch.autograd.grad(got, [leaf, weight_again], far(grad, 1))
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(grads, want_grads))
    with torch.no_grad():
        assert torch.equal(policy.causal_conv(leaf, weight, starts=starts), want)

"""The gated delta rule's precision before its outputs' rounding (``navi_amd.policy``).

Outputs of 16 bits hide what came before their rounding, unless one counts how many differ from
the exact result's rounding. An error e before the rounding changes a number whose neighbours
lie ulp apart with a chance of |e| / ulp, at most 1. With errors of the size that the float32
outputs are held to, 32 x 2^-24 of the root mean square, the expected share follows from the exact
numbers themselves.
"""

from __future__ import annotations

import pytest
import torch

from . import policy_reference as ref

pytestmark = pytest.mark.gpu

TOL = 32 * ref.EPS
FRACTION = {torch.bfloat16: 7, torch.float16: 10}  # bits of a number's fraction
LEAST = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -14}  # normal number


@pytest.fixture(scope="module")
def policy(gpu):
    from navi_amd import policy

    return policy


def make(envs, steps, hk, hv, kd, vd, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    unit = lambda x: torch.nn.functional.normalize(x, dim=-1)  # noqa: E731
    x = {"q": unit(rand(envs, steps, hk, kd)).to(dtype),
         "k": unit(rand(envs, steps, hk, kd) + 0.6 * rand(envs, 1, hk, kd)).to(dtype),
         "v": rand(envs, steps, hv, vd).to(dtype),
         "g": -torch.exp(rand(envs, steps, hv) * 1.5 - 3.0),
         "beta": torch.sigmoid(rand(envs, steps, hv) + 0.5)}
    return {n: t.cuda() for n, t in x.items()}, (0.3 * rand(envs, hv, kd, vd)).cuda()


def shares(got, want):
    """The share of ``got`` that is not the rounding of ``want``, and the share expected of errors of TOL."""
    dtype, want = got.dtype, want.detach()
    ulp = torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=LEAST[dtype]))) - FRACTION[dtype])
    error = TOL * float(want.square().mean().sqrt())
    return (float((got.detach().cpu() != want.to(dtype)).double().mean()),
            float((error / ulp).clamp(max=1.0).mean()))


@pytest.mark.parametrize("size", [(2, 300, 2, 2, 64, 64), (1, 200, 1, 2, 128, 128), (2, 150, 1, 1, 40, 72),
                                  (1, 1100, 1, 1, 64, 64)], ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_outputs_of_16_bits_are_rounded_once(policy, size, dtype):
    x, state = make(*size, dtype, seed=31)
    leaves = {n: t.clone().requires_grad_() for n, t in x.items()}
    o = policy.gated_delta_rule(*leaves.values(), initial_state=state)
    exact = {n: t.cpu().double().requires_grad_() for n, t in x.items()}
    want = ref.rule(*exact.values(), None, state, size[4] ** -0.5)[0]
    grad = torch.randn(o.shape, generator=torch.Generator().manual_seed(3)).to(dtype)
    names = ["q", "k", "v"]
    back = torch.autograd.grad(o, [leaves[n] for n in names], grad.cuda())
    back_want = torch.autograd.grad(want, [exact[n] for n in names], grad.double())
    for name, a, b in zip(["o", *names], [o, *back], [want, *back_want]):
        share, expected = shares(a, b)
        assert share <= expected, name


def test_float32_numbers_whose_low_bits_are_ones(policy):
    """One key and a start at every token: o = q k v and the state is k v of the last. A product is
    summed in float32 with its large term last, so a sum's rounding counts once (2^-23, however the
    sum rounds), and terms left out are held to 2^-26: 2.5 x 2^-24 a product, of which o has two
    and the state one."""
    steps, size = 70, 1 + 2.0 ** -7 - 2.0 ** -23
    one = torch.full((1, steps, 1, 1), size, device="cuda")
    v = one.expand(1, steps, 1, 32).contiguous()
    gate = torch.zeros(1, steps, 1, device="cuda")
    starts = torch.ones(1, steps, dtype=torch.bool, device="cuda")
    o, state = policy.gated_delta_rule(one, one, v, gate, torch.ones_like(gate), scale=1.0, starts=starts, return_state=True)
    assert float((o.double() / size ** 3 - 1).abs().max()) <= 6 * ref.EPS
    assert float((state.double() / size ** 2 - 1).abs().max()) <= 3 * ref.EPS

"""Orthogonalised updates (``navi_amd.policy.orthogonalize``) at the ends of their range on the GPU: wide matrices whose
size sits in a few numbers, factors at their limits.

Tolerances as in ``test_gpu_orthogonalize.py``: 2^-18 of the result's norm for products of two planes, 2^-10 for products
of one, and the result's own rounding.
"""

from __future__ import annotations

import pytest
import torch

from . import block_reference as ref
from .policy_reference import off

pytestmark = pytest.mark.gpu

FACTORS = (3.4445, -4.775, 2.0315)
TWO, ONE = 2.0 ** -18, 2.0 ** -10


@pytest.fixture(scope="module")
def policy(gpu):
    from navi_amd import policy

    return policy


def half_step(t):
    """A rounding of few numbers, half a step of each at most."""
    return 0.0 if t.dtype == torch.float32 else torch.finfo(t.dtype).eps / 2


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m, n", [(1, 1 << 19), (3, 1 << 20), (1 << 20, 2)])
def test_a_few_large_numbers_of_many(policy, m, n, out):
    """X's numbers then are near 1 whatever its length, and grow to 1.2 with its singular values."""
    g = torch.zeros(m, n)
    for i in range(min(m, n)):
        place = (i, 1000 + 7 * i) if m < n else (1000 + 7 * i, i)
        g[place] = 5.0 * 0.1 ** i
    want = ref.orthogonal(g, 5, FACTORS, 1e-6)
    to = torch.full((m, n), float("nan"), dtype=out, device="cuda")
    policy.orthogonalize([g.cuda()], out=[to])
    assert off(to, want) <= TWO + half_step(to)
    assert int(to.count_nonzero()) == min(m, n)


@pytest.mark.parametrize("out, products", [(torch.float32, TWO), (torch.bfloat16, ONE)])
def test_a_few_large_numbers_of_a_wide_matrix_with_many_rows(policy, out, products):
    rows, n = 300, 1 << 19
    small = torch.diag(torch.tensor([1.0] + [0.01] * (rows - 1)))
    columns = torch.arange(rows) * 1747 + 11
    g = torch.zeros(rows, n, device="cuda")
    g[:, columns.cuda()] = small.cuda()
    to = torch.empty(rows, n, dtype=out, device="cuda")
    policy.orthogonalize([g], out=[to])
    got = to[:, columns.cuda()]
    assert off(got, ref.orthogonal(small, 5, FACTORS, 1e-6)) <= products + half_step(to)
    assert int(to.count_nonzero()) == rows


@pytest.mark.parametrize("steps, factors", [(2, (7.8, 0.0, 0.0)), (1, (1.0, -60.0, 0.0)), (1, (-2.0, 0.0, 60.0)), (100, (1.5, -0.5, 0.0))])
def test_factors_at_their_limits(policy, steps, factors):
    """Singular values up to 7.9 between steps, and up to 62 of b A + c A A."""
    gen = torch.Generator().manual_seed(4)
    for m, n in ((5, 1 << 18), (40, 70)):
        g = torch.zeros(m, n)
        g[0, 3] = 1.0
        g[1:, 9:60] = 0.001 * torch.randn(m - 1, 51, generator=gen)
        want = ref.orthogonal(g, steps, factors, 0.0)
        x = g.cuda()
        policy.orthogonalize([x], steps=steps, factors=factors, eps=0.0)
        assert off(x, want) <= TWO

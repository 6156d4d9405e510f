"""What ``navi_amd.policy.orthogonalize`` loses before it rounds to bfloat16.

Matrices whose shorter side is up to 256 take products of two planes, 2^-18 of the result's norm after five steps
(``test_gpu_orthogonalize.py``). A number then rounds otherwise than the exact one where that lies within the error of
a border. Numbers of at least a tenth of the root mean square are at least 2^-8 / 10 of it apart from border to border:
2 x 2^-18 x 10 / 2^-8 = 2^-5.7 of them at most, were all so small; those of the mean's size one in 2^9. Products of one
plane leave 2^-12 to 2^-10: one number in 4 to one in 10.
"""

from __future__ import annotations

import pytest
import torch

from . import block_reference as ref
from .policy_reference import off
from .test_gpu_orthogonalize import FACTORS, PRODUCTS, momentum, policy  # noqa: F401

pytestmark = pytest.mark.gpu

SHORT = [(7, 256), (7, 2000), (2000, 7), (24, 24), (100, 100), (105, 256), (256, 256), (256, 2000), (1024, 256)]


@pytest.mark.parametrize("together", [False, True])
def test_short_matrices_are_rounded_once(policy, together):
    given = [momentum(m, n, torch.float32, seed=i) for i, (m, n) in enumerate(SHORT)]
    to = [torch.empty(g.shape, dtype=torch.bfloat16, device="cuda") for g in given]
    if together:  # (beside matrices that take one plane, in the middle of them)
        more = [momentum(1300, 1300, torch.float32, seed=20 + i) for i in range(8)]
        everything = [t for pair in zip(more, given) for t in pair] + given[8:]
        into = [t for pair in zip([torch.empty_like(t, dtype=torch.bfloat16) for t in more], to) for t in pair] + to[8:]
        policy.orthogonalize(everything, out=into)
    else:
        for g, o in zip(given, to):
            policy.orthogonalize([g], out=[o])
    for g, o in zip(given, to):
        want = ref.orthogonal(g, 5, FACTORS, 1e-6)
        large = want.abs() >= 0.1 * want.square().mean().sqrt()
        assert float((o.cpu() != want.to(torch.bfloat16))[large].double().mean()) <= 2.0 ** -6, tuple(g.shape)


@pytest.mark.parametrize("m, n", [(257, 257), (300, 520), (257, 4000)])
def test_longer_matrices_keep_their_bound(policy, m, n):
    g = momentum(m, n, torch.float32, seed=3)
    to = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    policy.orthogonalize([g], out=[to])
    assert off(to, ref.orthogonal(g, 5, FACTORS, 1e-6)) <= PRODUCTS[torch.bfloat16] + ref.rounding(to)


def test_results_do_not_depend_on_the_company_of_longer_matrices(policy):
    given = [momentum(m, n, torch.float32, seed=i) for i, (m, n) in enumerate([(64, 64), (300, 300), (128, 200), (520, 300)] * 4)]
    for dtype in (torch.bfloat16, torch.float32):
        to = [torch.empty(g.shape, dtype=dtype, device="cuda") for g in given]
        policy.orthogonalize(given, out=to)
        for g, o in zip(given, to):
            alone = torch.empty_like(o)
            policy.orthogonalize([g], out=[alone])
            assert torch.equal(alone, o)

"""Orthogonalised updates (``navi_amd.policy.orthogonalize``) on the GPU against the iteration in float64.

Tolerances. Five steps enlarge what a rounding leaves of the smallest singular values as they enlarge those
themselves (up to 3.4445^5 = 485 times), so errors are measured against the result's norm for matrices whose
singular values span less than that. Two planes hold 22 bits: a step rounds X, A and P to 2^-23 each and its
sums to a few 2^-24, less than 2^-20 together: 2^-18 after five steps that each turn over what came before.
One plane (bfloat16 results): 11 bits of A, P and the X in products, 2^-12 of each in the mean at most,
sums over many of them: 2^-10 over five steps, and the result's own rounding.
"""

from __future__ import annotations

import pytest
import torch

from . import block_reference as ref
from .policy_reference import off

pytestmark = pytest.mark.gpu

FACTORS = (3.4445, -4.775, 2.0315)
PRODUCTS = {torch.float32: 2.0 ** -18, torch.float16: 2.0 ** -18, torch.bfloat16: 2.0 ** -10}


def tolerance(t):
    return PRODUCTS[t.dtype] + ref.rounding(t)


@pytest.fixture(scope="module")
def policy(gpu):
    from navi_amd import policy

    return policy


def momentum(m, n, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    r = max(1, min(m, n) // 8)
    low = rand(m, r) * torch.exp(rand(r)) @ rand(r, n) / r ** 0.5
    return (1e-3 * (low + 0.5 * rand(m, n))).to(dtype).cuda()


SHAPES = [(1, 1), (1, 300), (300, 1), (7, 256), (256, 7), (128, 128), (129, 127), (105, 256), (64, 500), (600, 257), (33, 33)]


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_many_matrices_at_once(policy, dtype, out):
    given = [momentum(m, n, dtype, seed=i) for i, (m, n) in enumerate(SHAPES)]
    kept = [g.clone() for g in given]
    to = [torch.full(g.shape, float("nan"), dtype=out, device="cuda") for g in given]
    assert policy.orthogonalize(given, out=to) is None
    for g, k, o in zip(given, kept, to):
        assert torch.equal(g, k)
        assert off(o, ref.orthogonal(g, 5, FACTORS, 1e-6)) <= tolerance(o), tuple(g.shape)


def test_large_matrices_take_large_tiles(policy):
    """256 tiles of 256 x 256 and more go another way."""
    for dtype in (torch.bfloat16, torch.float32):
        given = [momentum(m, n, torch.float32, seed=i) for i, (m, n) in enumerate([(2000, 2100), (1030, 4000), (4000, 1030), (300, 260)])]
        given += [momentum(1500, 1500, torch.float32, seed=9), momentum(1500, 1500, torch.float32, seed=10)]
        to = [torch.empty(g.shape, dtype=dtype, device="cuda") for g in given]
        policy.orthogonalize(given, out=to)
        for g, o in zip(given, to):
            x = g.double()  # (on the GPU: the products are large)
            turned = x.shape[0] > x.shape[1]
            x = x.T.contiguous() if turned else x
            x = x / (x.norm() + 1e-6)
            for _ in range(5):
                gram = x @ x.T.contiguous()
                x = FACTORS[0] * x + (FACTORS[1] * gram + FACTORS[2] * (gram @ gram)) @ x
            assert off(o, (x.T if turned else x).cpu()) <= tolerance(o), tuple(g.shape)


def test_singular_values_come_out_near_one(policy):
    for shape in ((96, 96), (300, 80)):
        u, _, v = torch.linalg.svd(torch.randn(*shape, generator=torch.Generator().manual_seed(1)), full_matrices=False)
        s = torch.logspace(0, -1, min(shape))
        x = ((u * s) @ v).cuda()
        policy.orthogonalize([x])
        got = torch.linalg.svdvals(x.cpu().double())
        assert float(got.min()) > 0.6 and float(got.max()) < 1.3
        # (the polynomial of the singular values, in float64)
        want = s.double() / s.double().norm()
        for _ in range(5):
            want = FACTORS[0] * want + FACTORS[1] * want ** 3 + FACTORS[2] * want ** 5
        assert off(got, want.sort(descending=True).values) <= 2.0 ** -18


@pytest.mark.parametrize("steps, factors", [(1, FACTORS), (2, (1.5, -0.5, 0.0)), (9, (1.875, -1.25, 0.375))])
def test_other_polynomials(policy, steps, factors):
    x = momentum(150, 90, torch.float32, seed=3)
    want = ref.orthogonal(x, steps, factors, 1e-3)
    policy.orthogonalize([x], steps=steps, factors=factors, eps=1e-3)
    assert off(x, want) <= 2.0 ** -18


def test_in_place_strides_and_nothing_else_is_written(policy):
    plain = [momentum(m, n, torch.float32, seed=i) for i, (m, n) in enumerate([(100, 150), (150, 100), (40, 40)])]
    want = [x.clone() for x in plain]
    policy.orthogonalize(want)
    for column in (0, 1):  # of a wider array; transposed
        arrays = [torch.full((x.shape[0] + 6, x.shape[1] + 9), 3.0, device="cuda") for x in plain]
        views = [a[3:-3, 5:-4] for a in arrays]
        if column:
            arrays = [torch.full((x.shape[1] + 6, x.shape[0] + 9), 3.0, device="cuda") for x in plain]
            views = [a[3:-3, 5:-4].T for a in arrays]
        for v, x in zip(views, plain):
            v.copy_(x)
        into = [torch.empty(x.shape, device="cuda") for x in plain]
        policy.orthogonalize(views, out=into)
        policy.orthogonalize(views)
        for a, v, w, i in zip(arrays, views, want, into):
            # (sums over the squares go along other axes: the last bits may differ)
            assert off(v, w.cpu().double()) <= 2.0 ** -18 and torch.equal(v, i)
            border = a.clone()
            border[3:-3, 5:-4] = 3.0
            assert (border == 3.0).all()
    every_other = torch.zeros(100, 300, device="cuda")
    policy.orthogonalize([plain[0]], out=[every_other[:, ::2]])
    assert torch.equal(every_other[:, ::2], want[0]) and not every_other[:, 1::2].any()


def test_zeros_none_and_empty_matrices(policy):
    x = [torch.zeros(50, 60, device="cuda"), None, torch.zeros(0, 5, device="cuda"), momentum(20, 30, torch.float32)]
    want = ref.orthogonal(x[3], 5, FACTORS, 1e-6)
    policy.orthogonalize(x)
    assert not x[0].any() and off(x[3], want) <= PRODUCTS[torch.float32]


def test_numbers_of_any_size(policy):
    for scale in (1e-30, 1e-12, 1e18, 1e30):
        x = torch.randn(90, 70, generator=torch.Generator().manual_seed(2)).cuda() * scale
        want = ref.orthogonal(x, 5, FACTORS, 0.0)
        policy.orthogonalize([x], eps=0.0)
        assert off(x, want) <= PRODUCTS[torch.float32], scale
    one = torch.zeros(40, 70, device="cuda")
    one[3, 5] = 7.0  # (a single number: all of X's size in one place)
    want = ref.orthogonal(one, 5, FACTORS, 1e-6)
    policy.orthogonalize([one])
    assert off(one, want) <= PRODUCTS[torch.float32]


def test_results_do_not_depend_on_the_company(policy):
    x = [momentum(m, n, torch.bfloat16, seed=i) for i, (m, n) in enumerate([(128, 200), (200, 128), (64, 64)] * 15)]
    alone = [t.clone() for t in x]
    for t in alone:
        policy.orthogonalize([t])
    policy.orthogonalize(x)
    assert all(torch.equal(a, b) for a, b in zip(x, alone))

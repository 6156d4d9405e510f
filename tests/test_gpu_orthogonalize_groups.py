"""Calls of ``navi_amd.policy.orthogonalize`` that one set of launches does not hold: more matrices than a launch names,
results of several types in turn, more workspace than matrices share. Each matrix comes out as it does alone."""

from __future__ import annotations

import pytest
import torch

from . import block_reference as ref
from .policy_reference import off
from .test_gpu_orthogonalize import FACTORS, momentum, policy, tolerance  # noqa: F401

pytestmark = pytest.mark.gpu

TYPES = (torch.bfloat16, torch.float32, torch.float16)
SHAPES = [(20, 30), (64, 64), (65, 33), (1, 100), (100, 3), (30, 80)]


def alone(policy, given, like):
    to = torch.empty_like(like)
    policy.orthogonalize([given], out=[to])
    return to


@pytest.mark.parametrize("count", [61, 62, 63, 130])
def test_more_matrices_than_a_launch_names(policy, count):
    given = [momentum(*SHAPES[i % 6], TYPES[i % 2], seed=i) for i in range(count)]
    for dtype in TYPES:
        to = [torch.full(g.shape, float("nan"), dtype=dtype, device="cuda") for g in given]
        policy.orthogonalize(given, out=to)
        for i, (g, o) in enumerate(zip(given, to)):
            assert torch.equal(o, alone(policy, g, o)), i
            assert off(o, ref.orthogonal(g, 5, FACTORS, 1e-6)) <= tolerance(o), i


@pytest.mark.parametrize("run", [1, 2, 7])
def test_results_of_several_types_in_turn(policy, run):
    """Types change every `run` matrices, with empty ones and None where they do."""
    given, to = [], []
    for i in range(70):
        if i % run == 0:
            given += [None, torch.zeros(0, 9, device="cuda")]
            to += [None, torch.zeros(0, 9, device="cuda", dtype=TYPES[i // run % 3])]
        given.append(momentum(*SHAPES[i % 6], TYPES[i % 3], seed=i))
        to.append(torch.full(given[-1].shape, float("nan"), dtype=TYPES[i // run % 3], device="cuda"))
    policy.orthogonalize(given, out=to)
    for i, (g, o) in enumerate(zip(given, to)):
        if g is not None and g.numel():
            assert torch.equal(o, alone(policy, g, o)), i
            assert off(o, ref.orthogonal(g, 5, FACTORS, 1e-6)) <= tolerance(o), i
    kept = [None if g is None else g.clone() for g in given]
    policy.orthogonalize(given)  # (in their own places, each in its own type)
    for i, (g, k) in enumerate(zip(given, kept)):
        if g is not None and g.numel():
            assert torch.equal(g, alone(policy, k, g)), i


def test_more_workspace_than_matrices_share(policy):
    """Three matrices of 3 GiB of workspace each: one after the other.

    A's sums over 2^20 numbers are 3 x 2^16 additions of float32 one after the other (16 numbers each, three products
    of planes), that round to half a step of the sum so far, 2^-24 of the whole at most, with either sign: in all
    2^-24 sqrt(3 x 2^16) = 2^-15.2 of it, beside 2^-18 as for short ones."""
    given = [1e-3 * torch.randn(256, 1 << 20, device="cuda", generator=torch.Generator(device="cuda").manual_seed(i)) for i in range(3)]
    to = [torch.empty_like(g) for g in given]
    policy.orthogonalize(given, out=to)
    for g, o in zip(given, to):
        assert torch.equal(o, alone(policy, g, o))
        x = g.double()
        x /= x.norm() + 1e-6
        # (the products' sums are 256 x 256 polynomials of the first: X = q(G G^T) G)
        whole, gram = torch.eye(256, dtype=torch.float64, device="cuda"), x @ x.T.contiguous()
        for _ in range(5):
            now = whole @ gram @ whole.T.contiguous()
            whole = FACTORS[0] * whole + (FACTORS[1] * now + FACTORS[2] * now @ now) @ whole
        assert off(o, (whole @ x).cpu()) <= tolerance(o) + 2.0 ** -24 * (3 * 2 ** 16) ** 0.5


@pytest.mark.parametrize("dtype", TYPES)
def test_small_matrices_in_large_company(policy, dtype):
    """Tiles are those of the call's large matrices."""
    given = [momentum(m, n, torch.float32, seed=i) for i, (m, n) in enumerate([(7, 4096), (200, 90), (300, 520)])]
    given.insert(1, momentum(4096, 4100, torch.float32, seed=50))
    to = [torch.empty(g.shape, dtype=dtype, device="cuda") for g in given]
    policy.orthogonalize(given, out=to)
    for g, o in zip(given, to):
        if g.shape[0] < 4096:
            assert off(o, ref.orthogonal(g, 5, FACTORS, 1e-6)) <= tolerance(o), tuple(g.shape)

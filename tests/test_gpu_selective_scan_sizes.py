"""The selective scan's gradients where keys lie on both sides of 64, in one launch and in two, and the ends of its ranges.

Keys of the gradients' scans have state_dim and head_dim numbers; those of up to 64 and of up to 128 go in launches of
their own, unless the card holds all workgroups of 128 at once (512 of 16 bits of one plane, 256 otherwise): then all go
in one. Tolerances as in ``test_gpu_selective_scan.py``.
"""

from __future__ import annotations

import pytest
import torch

from .test_gpu_selective_scan import TOL, call, compare, make, off, policy, reference, tolerance  # noqa: F401

pytestmark = pytest.mark.gpu

LARGE = [  # envs, steps, heads, groups, state_dim, head_dim: more workgroups than the card holds at once
    (70, 130, 4, 2, 128, 48, torch.bfloat16),
    (70, 130, 4, 2, 48, 128, torch.bfloat16),
    (70, 66, 4, 1, 72, 40, torch.float32),
    (70, 66, 4, 4, 40, 72, torch.float16),
]


@pytest.mark.parametrize("with_state", [False, True])
@pytest.mark.parametrize("size", LARGE, ids=str)
def test_keys_on_both_sides_of_64_in_launches_of_their_own(policy, size, with_state):
    x, state, starts = make(*size, seed=31)
    compare(policy, size, x, state if with_state else None, starts)


@pytest.mark.parametrize("envs, dtype", [(128, torch.bfloat16), (129, torch.bfloat16), (64, torch.float32), (65, torch.float32)], ids=str)
def test_on_either_side_of_what_the_card_holds(policy, envs, dtype):
    """Two blocks of 40 x 72 and two of 72 x 40 a head: 4 x 128 or 4 x 64 workgroups, or one head more."""
    size = (envs, 70, 1, 1, 40, 72, dtype)
    x, _, starts = make(*size, seed=32)
    compare(policy, size, x, None, starts)


def test_long_walks_with_keys_on_both_sides_of_64(policy):
    """Segments in launches of their own for each: 30 heads of four blocks in 5 segments."""
    size = (30, 64 * 12 + 7, 1, 1, 24, 100, torch.float32)
    x, state, starts = make(*size, seed=33, often=0.003)
    x["dt"] -= 3.0  # (a state that lasts through segments)
    compare(policy, size, x, state, starts)


def test_as_many_heads_as_there_may_be(policy):
    size = (2, 67, 16384, 64, 3, 2, torch.bfloat16)
    x, state, starts = make(*size, seed=34)
    compare(policy, size, x, state, starts)
    y = call(policy, {n: t[:, :1] if t.dim() > 1 else t for n, t in x.items()})
    assert off(y, reference({n: t[:, :1] if t.dim() > 1 else t for n, t in x.items()}, None, None)[0]) <= tolerance(y)

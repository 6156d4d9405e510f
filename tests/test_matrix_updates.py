"""Which parameters ``navi_amd.memory_policy.MatrixUpdates`` takes as matrices (no GPU: nothing is stepped here), and what
it does to a policy's convolutions."""

from __future__ import annotations

import pytest
import torch

from navi_amd import memory_policy as mp

SMALL = dict(inputs=24, width=32, heads=4, head_dim=8, groups=2, state_dim=16, taps=3, blocks=2)


def names_of(model, parameters):
    names = {id(p): n for n, p in model.named_parameters()}
    return {names[id(p)] for p in parameters}


def test_taps_are_no_matrices():
    """A convolution's taps are a filter a channel, not a linear map of channels."""
    model = mp.SelectivePolicy(**SMALL, device="cpu")
    optimizer = mp.MatrixUpdates.of(model, lr=1e-3)
    taps = {n for n, _ in model.named_parameters() if n.endswith("taps_weight")}
    assert len(taps) == 2
    adams = names_of(model, optimizer.adam.param_groups[0]["params"])
    matrices = names_of(model, optimizer.matrices)
    assert taps <= adams and not taps & matrices
    assert matrices | adams == {n for n, _ in model.named_parameters()}
    assert matrices == {n for n, _ in model.named_parameters() if n.endswith(("project.weight", "steps.weight", "merge.weight", "encode.weight", "predict.weight"))}


def test_policies_without_filters():
    model = mp.MemoryPolicy(device="cpu")
    optimizer = mp.MatrixUpdates.of(model, lr=1e-3)
    assert names_of(model, optimizer.matrices) == {n for n, p in model.named_parameters() if p.dim() == 2}


def test_filters_that_are_no_parameters_are_refused():
    p = torch.nn.Parameter(torch.zeros(4, 3))
    with pytest.raises(ValueError, match="filters"):
        mp.MatrixUpdates([p], filters=[torch.nn.Parameter(torch.zeros(4, 3))])
    assert mp.MatrixUpdates([p], filters=[p]).matrices == []


@pytest.mark.gpu
def test_taps_are_stepped_by_adam(gpu):
    torch.manual_seed(0)
    model = mp.SelectivePolicy(**SMALL, dtype=torch.float32)
    stepper = mp.OPTIMIZERS["orthogonal"](model, lr=1e-2)
    twins = [torch.nn.Parameter(block.taps_weight.detach().clone()) for block in model.blocks]
    adam = torch.optim.Adam(twins, lr=1e-2)
    for _ in range(2):
        model(torch.randn(3, 20, 24, device="cuda"), torch.zeros(3, 20, dtype=torch.bool, device="cuda")).square().mean().backward()
        for twin, block in zip(twins, model.blocks):
            twin.grad = block.taps_weight.grad.clone()
        stepper.step()
        adam.step()
        stepper.zero_grad()
    for twin, block in zip(twins, model.blocks):
        assert torch.equal(twin, block.taps_weight)

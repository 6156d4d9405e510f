"""The example that runs the policy's operators together (``navi_amd.memory_policy``): acting and
learning give the same numbers, and training on a room's frames lowers the loss."""

from __future__ import annotations

import json

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_acting_and_learning_agree_and_train(gpu, dtype):
    from navi_amd import memory_policy as mp
    from navi_amd import scenes as S

    room = S.box_room()
    got = mp.run([(room.compile(), room.bbox_min, room.bbox_max)], actors=6, steps=70, updates=4, azimuth_bins=64,
                 elevation_bins=16, max_distance=30.0, sdf_max_steps=64, seed=3, dtype=dtype)
    # float32: sums in other orders through five products; bfloat16: the memory's inputs are the
    # same roundings of nearly the same numbers, a unit of which is 2^-8
    assert got["acted_against_learned"] <= (1e-4 if dtype == torch.float32 else 2.0 ** -7)
    assert got["episodes"] >= 6
    assert got["loss_last"] < 0.5 * got["loss_first"]
    assert got["grad_norm_first"] > 0.0


def test_gradients_through_the_operators(gpu):
    """The example's gradients against the same policy with the recurrence in plain float64."""
    from navi_amd import memory_policy as mp

    from . import policy_reference as ref

    torch.manual_seed(0)
    model = mp.MemoryPolicy(inputs=24, width=32, heads=2, head_dim=16, rotary=8, positions=128, dtype=torch.float32)
    x = torch.randn(3, 80, 24, device="cuda")
    starts = torch.rand(3, 80, device="cuda") < 0.05
    positions = torch.arange(80, device="cuda", dtype=torch.int32).expand(3, 80).contiguous()
    state = 0.1 * torch.randn(3, 2, 16, 16, device="cuda")
    loss = model(x, starts, positions, state).square().mean()
    grads = dict(zip([n for n, _ in model.named_parameters()], torch.autograd.grad(loss, list(model.parameters()))))

    plain = {n: p.detach().cpu().double().requires_grad_() for n, p in model.named_parameters()}
    h = torch.nn.functional.gelu(x.cpu().double() @ plain["encode.weight"].T + plain["encode.bias"])
    q, k, v = (h @ plain["project.weight"].T).unflatten(-1, (6, 16)).chunk(3, dim=2)
    q, k = (_norm(t, model, positions) for t in (q, k))
    decay, write = (h @ plain["gates.weight"].T + plain["gates.bias"]).chunk(2, dim=-1)
    o, _ = _rule(ref, q, k, v, -0.2 * torch.nn.functional.softplus(decay), torch.sigmoid(write), starts, state)
    said = (h + o.flatten(-2) @ plain["merge.weight"].T) @ plain["predict.weight"].T + plain["predict.bias"]
    want_loss = said.square().mean()
    want = torch.autograd.grad(want_loss, list(plain.values()))
    assert abs(float(loss.detach()) - float(want_loss.detach())) <= 1e-5 * float(want_loss.detach())
    for n, w in zip(plain, want):
        assert ref.off(grads[n], w) <= 1e-4, n  # (float32 products of the library around the operators)


def _norm(x, model, positions):
    y = x / torch.sqrt(x.square().sum(-1, keepdim=True) + 1e-6)
    at = positions.cpu().long()
    c, s = (z.cpu().double()[at][:, :, None] for z in (model.cos, model.sin))
    a, b = y[..., :4], y[..., 4:8]
    return torch.cat([a * c - b * s, b * c + a * s, y[..., 8:]], -1)


def _rule(ref, q, k, v, g, beta, starts, state):
    return ref.rule(q, k, v, g, beta, starts, state, 16 ** -0.5)


def test_the_command(gpu, capsys):
    from navi_amd import memory_policy as mp

    assert mp.main(["--actors", "4", "--steps", "20", "--updates", "2", "--azimuth-bins", "64", "--elevation-bins", "16",
                    "--json"]) == 0
    out = json.loads(capsys.readouterr().out)
    assert out["actors"] == 4 and out["learn_ms"] > 0 and out["act_ms"] > 0

"""The example's policy with blocks of a selective scan (``navi_amd.memory_policy``): the block's operators together,
acting and learning, their gradients, and updates by orthogonalised momenta."""

from __future__ import annotations

import json

import pytest
import torch

from . import block_reference as ref
from .policy_reference import off

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("core", ["selective", "delta"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_acting_and_learning_agree(gpu, dtype, core):
    from navi_amd import memory_policy as mp
    from navi_amd import scenes as S

    room = S.box_room()
    got = mp.run([(room.compile(), room.bbox_min, room.bbox_max)], actors=6, steps=70, updates=3, azimuth_bins=64,
                 elevation_bins=16, max_distance=30.0, sdf_max_steps=64, seed=3, dtype=dtype, core=core, optimizer="orthogonal")
    # float32: sums in other orders through the blocks' products; bfloat16: the same roundings of nearly the same
    # numbers, a unit of which is 2^-8
    assert got["acted_against_learned"] <= (1e-4 if dtype == torch.float32 else 2.0 ** -7)
    assert got["episodes"] >= 6 and got["grad_norm_first"] > 0.0


def test_gradients_through_the_blocks(gpu):
    """The example's output and gradients against the same policy in plain float64."""
    from navi_amd import memory_policy as mp

    torch.manual_seed(0)
    model = mp.SelectivePolicy(inputs=24, width=32, heads=4, head_dim=8, groups=2, state_dim=16, taps=3, blocks=2, dtype=torch.float32)
    x = torch.randn(3, 80, 24, device="cuda")
    starts = torch.rand(3, 80, device="cuda") < 0.05
    state = tuple(0.3 * torch.randn_like(t) for t in model.initial_state(3))
    said = model(x, starts, None, state)
    loss = said.square().mean()
    grads = dict(zip([n for n, _ in model.named_parameters()], torch.autograd.grad(loss, list(model.parameters()))))

    plain = {n: p.detach().cpu().double().requires_grad_() for n, p in model.named_parameters()}
    stream = torch.nn.functional.gelu(x.cpu().double() @ plain["encode.weight"].T + plain["encode.bias"])
    normed = stream
    for i in range(2):
        p = {n.split(".", 2)[2]: t for n, t in plain.items() if n.startswith(f"blocks.{i}.")}
        taken, gate = (normed @ p["project.weight"].T).split((96, 32), -1)
        taken, _ = ref.conv(taken, p["taps_weight"], p["taps_bias"], starts, state[2 * i], "silu")
        xs, b, c = taken.split((32, 32, 32), -1)
        o, _ = ref.scan(xs.unflatten(-1, (4, 8)), normed @ p["steps.weight"].T, -p["rate"].abs(), b.unflatten(-1, (2, 16)),
                        c.unflatten(-1, (2, 16)), p["skip"], p["step_bias"], starts, state[2 * i + 1])
        stream, normed = ref.block(o.flatten(-2) @ p["merge.weight"].T, stream, gate, p["scale"], p["post"], p["pre"], 1e-6)
    want_said = normed @ plain["predict.weight"].T + plain["predict.bias"]
    want = torch.autograd.grad(want_said.square().mean(), list(plain.values()))
    assert off(said, want_said) <= 1e-5
    for n, w in zip(plain, want):
        assert off(grads[n], w) <= 1e-4, n  # (float32 products of the library around the operators)


def test_frames_one_by_one_are_a_rollout(gpu):
    """Acting carries windows and states on as a rollout does, over episode starts and from one rollout to the next."""
    from navi_amd import memory_policy as mp

    torch.manual_seed(1)
    model = mp.SelectivePolicy(inputs=24, width=64, heads=2, head_dim=32, state_dim=16, blocks=2, dtype=torch.float32)
    x = torch.randn(5, 40, 24, device="cuda")
    starts = torch.rand(5, 40, device="cuda") < 0.1
    state = model.initial_state(5)
    acted = torch.stack([model.act(x[:, t], starts[:, t], None, state) for t in range(40)], 1)
    with torch.no_grad():
        whole = model(x, starts, None, model.initial_state(5))
        begun = model(x, starts, None, None)
    # float32 products in other orders, two blocks: a few 2^-24 of each of some twenty sums, that norms keep in size
    assert off(acted, whole.cpu().double()) <= 1e-5 and torch.equal(whole, begun)
    again = model.initial_state(5)
    for t in range(20):
        model.act(x[:, t], starts[:, t], None, again)
    with torch.no_grad():
        assert off(model(x[:, 20:], starts[:, 20:], None, again), whole[:, 20:].cpu().double()) <= 1e-5


def test_matrix_updates(gpu):
    """Matrices move along their orthogonalised momenta, other parameters as by Adam, what has no gradient stays."""
    from navi_amd import memory_policy as mp

    torch.manual_seed(2)
    shapes = [(48, 96), (96, 48), (64, 64), (5, 7)]
    matrices = [torch.nn.Parameter(torch.randn(s, device="cuda")) for s in shapes]
    vectors = [torch.nn.Parameter(torch.randn(9, device="cuda")) for _ in range(2)]
    optimizer = mp.MatrixUpdates([*matrices, *vectors], lr=0.5, momentum=0.75)
    twins = [torch.nn.Parameter(v.detach().clone()) for v in vectors]
    adam = torch.optim.Adam(twins, lr=0.5)
    held = [torch.zeros(s, dtype=torch.float64) for s in shapes]
    for step in range(3):
        for p in matrices + vectors:
            p.grad = torch.randn_like(p)
        for v, t in zip(vectors, twins):
            t.grad = v.grad.clone()
        matrices[3].grad = None
        before = [p.detach().clone() for p in matrices]
        optimizer.step()
        adam.step()
        assert all(torch.equal(v, t) for v, t in zip(vectors, twins))
        assert torch.equal(matrices[3], before[3])
        for p, b, h in list(zip(matrices, before, held))[:3]:
            h.lerp_(p.grad.cpu().double(), 0.25)
            want = -0.2 * 0.5 * max(p.shape) ** 0.5 * ref.orthogonal(h, 5, (3.4445, -4.775, 2.0315), 1e-6)
            # products of one float16 each (2^-10 over five steps), the update's own rounding, and sums with weights of
            # some ten times its size in float32
            assert off(p - b, want) <= 2.0 ** -10 + 2.0 ** -9 + 2.0 ** -19, step
    optimizer.zero_grad()
    assert all(p.grad is None for p in matrices + vectors)


@pytest.mark.parametrize("optimizer", ["adam", "orthogonal"])
def test_the_command(gpu, capsys, optimizer):
    from navi_amd import memory_policy as mp

    assert mp.main(["--actors", "4", "--steps", "20", "--updates", "2", "--azimuth-bins", "64", "--elevation-bins", "16",
                    "--core", "selective", "--optimizer", optimizer, "--json"]) == 0
    out = json.loads(capsys.readouterr().out)
    assert out["core"] == "selective" and out["optimizer"] == optimizer and out["learn_ms"] > 0 and out["act_ms"] > 0

"""The example's rollouts (``navi_amd.memory_policy.collect``) without a GPU: a harness whose frames
and collisions are known."""

from __future__ import annotations

import pytest
import torch

pytest.importorskip("navi_amd._policy_native")
from navi_amd import memory_policy as mp  # noqa: E402

ACTORS, STEPS = 3, 5
INPUTS = mp.POOL[0] * mp.POOL[1]


class Harness:
    """Frame n (from 1 on) shows n; ``collides[a]`` are the frames in which actor a collides."""

    def __init__(self, collides):
        self.collides, self.n = collides, 0
        self.obs = torch.zeros(ACTORS, 3, *mp.POOL)
        self.collision = torch.zeros(ACTORS, dtype=torch.int32)

    def step(self):
        self.n += 1
        self.obs.fill_(self.n + 0.5)
        self.collision.copy_(torch.tensor([int(self.n in c) for c in self.collides]))


class Model:
    """Acts by what it has seen: the state holds a count of frames since the episode's start."""

    def __init__(self):
        self.acted = []

    def act(self, x, starts, positions, state):
        state.masked_fill_(starts[:, None], 0.0)
        state += 1
        self.acted.append((x[:, 0].clone(), starts.clone(), positions.clone(), state[:, 0].clone()))
        return x


def collected(rollouts, collides):
    harness, model = Harness(collides), Model()
    rollout = mp.Rollout(ACTORS, STEPS, INPUTS, "cpu")
    state = torch.full((ACTORS, 1), 100.0)
    starts, positions = torch.ones(ACTORS, dtype=torch.bool), torch.zeros(ACTORS, dtype=torch.int32)
    kept = []
    for _ in range(rollouts):
        mp.collect(harness, model, rollout, state, starts, positions)
        kept.append((rollout.frames[:, :, 0].clone(), rollout.starts.clone(), rollout.positions.clone(),
                     rollout.state.clone(), rollout.acted[:, :, 0].clone()))
    return harness, model, kept


def test_frames_follow_each_other_over_rollouts():
    harness, model, kept = collected(3, [()] * ACTORS)
    assert [int(x[0]) for x, *_ in model.acted] == list(range(1, 3 * STEPS + 1))  # each frame acted on, once
    assert harness.n == 3 * STEPS + 1
    for i, (frames, _, positions, state, acted) in enumerate(kept):
        first = i * STEPS
        assert frames[0].tolist() == [first + 1.0 + n for n in range(STEPS + 1)]
        assert positions[0].tolist() == [first + n for n in range(STEPS + 1)]
        assert acted[0].tolist() == frames[0, :-1].tolist()
        assert float(state[0]) == (first if i else 100.0)  # before the rollout's first frame


@pytest.mark.parametrize("frame", [1, 3, STEPS, STEPS + 1, STEPS + 2, 2 * STEPS, 2 * STEPS + 1])
def test_a_collision_begins_an_episode(frame):
    """The frame after the one in which an actor collides is the first of a new episode, wherever in a
    rollout that is; the other actors go on."""
    _, model, kept = collected(3, [(), (frame,), ()])
    for n, (x, starts, positions, seen) in enumerate(model.acted, 1):
        assert starts.tolist() == [n == 1, n in (1, frame + 1), n == 1]
        place = n - 1 if n <= frame else n - 1 - frame
        assert positions.tolist() == [n - 1, place, n - 1]
        assert seen.tolist() == [n, place + 1, n]
    for i, (frames, starts, positions, *_) in enumerate(kept):
        for t in range(STEPS + 1):
            n = i * STEPS + t + 1
            assert frames[1, t] == n
            assert bool(starts[1, t]) == (n in (1, frame + 1))
            assert int(positions[1, t]) == (n - 1 if n <= frame else n - 1 - frame)

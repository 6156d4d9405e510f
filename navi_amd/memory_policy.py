"""A policy with a memory over the tracer's observations: acting frame by frame, learning over
rollouts. An example of ``navi_amd.policy`` as a trainer uses it, and a command that runs it::

    python -m navi_amd.memory_policy [--gmdag-file a.gmdag ...] --actors 64 --steps 128 --json

The reference's actor (``projects/actor``) encodes the ``(B, 3, Az, El)`` observation, passes it
through a temporal core and trains on rollouts of its in-process backend. ``MemoryPolicy`` is
such a core, small: pooled log-depth, one gated delta memory per head whose queries and keys
are normed and rotated by the step's place in its episode, and a head that predicts the next
frame (what the command trains on: the tracer alone has no rewards). Each update of the
command is one rollout of every actor, traced by ``bench_sdfdag``'s harness: while acting,
``gated_delta_step`` carries a state per actor, an actor that collides begins a new episode;
then ``gated_delta_rule`` reads the whole rollout with gradients, from the state at its
beginning, and ``clip_grad_norm`` bounds the update.
"""

from __future__ import annotations

import argparse
import json
import sys
import time
from pathlib import Path
from typing import Any

import torch
import torch.nn.functional as F

from . import policy

POOL = (32, 6)  # azimuth and elevation cells of a frame's features


def features(depth: torch.Tensor) -> torch.Tensor:
    """``[Actors, Az, El]`` log-normalised depth -> ``[Actors, 192]`` cell means, about zero."""
    return F.adaptive_avg_pool2d(depth[:, None], POOL).flatten(1) - 0.5


class MemoryPolicy(torch.nn.Module):
    """``act`` for one frame of every actor, ``forward`` for rollouts; the same numbers."""

    def __init__(self, inputs: int = POOL[0] * POOL[1], width: int = 256, heads: int = 4, head_dim: int = 64,
                 rotary: int = 32, positions: int = 4096, dtype: torch.dtype = torch.bfloat16, device="cuda") -> None:
        super().__init__()
        self.heads, self.head_dim, self.dtype = heads, head_dim, dtype
        inner = heads * head_dim
        self.encode = torch.nn.Linear(inputs, width, device=device)
        self.project = torch.nn.Linear(width, 3 * inner, bias=False, device=device)
        self.gates = torch.nn.Linear(width, 2 * heads, device=device)
        self.merge = torch.nn.Linear(inner, width, bias=False, device=device)
        self.predict = torch.nn.Linear(width, inputs, device=device)
        angle = torch.arange(positions, device=device)[:, None] * 10000.0 ** (
            -torch.arange(rotary // 2, device=device) / (rotary // 2))
        self.register_buffer("cos", torch.cos(angle))
        self.register_buffer("sin", torch.sin(angle))

    def initial_state(self, actors: int) -> torch.Tensor:
        return torch.zeros(actors, self.heads, self.head_dim, self.head_dim, device=self.cos.device)

    def _inputs(self, x: torch.Tensor, positions: torch.Tensor):
        """q, k, v, g, beta of features ``[Actors, Steps, Inputs]``, and the residual stream."""
        h = F.gelu(self.encode(x))
        # views of one projection: the operators read them where they are
        q, k, v = self.project(h).to(self.dtype).unflatten(-1, (3 * self.heads, self.head_dim)).chunk(3, dim=2)
        q, k = policy.qk_norm(q, k, norm="l2", cos=self.cos, sin=self.sin, positions=positions)
        decay, write = self.gates(h).chunk(2, dim=-1)
        return q, k, v, -0.2 * F.softplus(decay), torch.sigmoid(write), h

    def _output(self, o: torch.Tensor, h: torch.Tensor) -> torch.Tensor:
        return self.predict(h + self.merge(o.flatten(-2).float()))

    def forward(self, x, starts, positions, state=None):
        """Rollouts: ``x`` ``[Actors, Steps, Inputs]``, ``starts`` bool and ``positions`` int32
        ``[Actors, Steps]``, the memory's ``state`` before them. Predicts each next frame."""
        q, k, v, g, beta, h = self._inputs(x, positions)
        return self._output(policy.gated_delta_rule(q, k, v, g, beta, starts=starts, initial_state=state), h)

    @torch.no_grad()
    def act(self, x, starts, positions, state):
        """One frame: ``x`` ``[Actors, Inputs]``, ``starts`` and ``positions`` ``[Actors]``;
        ``state`` is updated in place."""
        q, k, v, g, beta, h = (t.squeeze(1) for t in self._inputs(x[:, None], positions[:, None]))
        return self._output(policy.gated_delta_step(q, k, v, g, beta, state, starts=starts), h)


class Rollout:
    """One rollout's frames, episode starts and places, and the state before it (None before the first)."""

    def __init__(self, actors: int, steps: int, inputs: int, device) -> None:
        self.frames = torch.empty(actors, steps + 1, inputs, device=device)
        self.starts = torch.zeros(actors, steps + 1, dtype=torch.bool, device=device)
        self.positions = torch.zeros(actors, steps + 1, dtype=torch.int32, device=device)
        self.acted = torch.empty(actors, steps, inputs, device=device)
        self.state: torch.Tensor | None = None


def collect(harness, model: MemoryPolicy, rollout: Rollout, state: torch.Tensor, starts: torch.Tensor,
            positions: torch.Tensor) -> None:
    """Steps every actor through a rollout; ``state`` (before the rollout's last frame), ``starts`` and
    ``positions`` (of that frame) are carried on in place. The last frame is only predicted: the next
    rollout begins with it."""
    steps = rollout.acted.shape[1]
    if rollout.state is None:
        harness.step()
        rollout.frames[:, 0] = features(harness.obs[:, 0])
    else:
        rollout.frames[:, 0] = rollout.frames[:, steps]
    rollout.state = state.clone()
    rollout.starts[:, 0], rollout.positions[:, 0] = starts, positions
    for t in range(steps):
        rollout.acted[:, t] = model.act(rollout.frames[:, t], starts, positions, state)
        starts.copy_(harness.collision != 0)  # in frame t: the next one begins an episode
        positions.add_(1).masked_fill_(starts, 0)
        harness.step()
        rollout.frames[:, t + 1] = features(harness.obs[:, 0])
        rollout.starts[:, t + 1], rollout.positions[:, t + 1] = starts, positions


def learn(model: MemoryPolicy, optimizer, rollout: Rollout, max_norm: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """One update over a rollout: (loss, gradient norm, predictions)."""
    said = model(rollout.frames[:, :-1], rollout.starts[:, :-1], rollout.positions[:, :-1], rollout.state)
    same = ~rollout.starts[:, 1:, None]  # the next frame belongs to the episode
    loss = ((said - rollout.frames[:, 1:]).square() * same).sum() / same.sum().clamp(min=1) / said.shape[-1]
    optimizer.zero_grad(set_to_none=True)
    loss.backward()
    norm = policy.clip_grad_norm([p.grad for p in model.parameters()], max_norm)
    optimizer.step()
    return loss.detach(), norm, said.detach()


def run(scenes, *, actors: int, steps: int, updates: int, azimuth_bins: int, elevation_bins: int, max_distance: float,
        sdf_max_steps: int, seed: int, max_norm: float = 1.0, dtype: torch.dtype = torch.bfloat16) -> dict[str, Any]:
    from .bench_sdfdag import ObservationHarness

    torch.manual_seed(seed)
    harness = ObservationHarness(scenes, actors, azimuth_bins, elevation_bins, max_distance, sdf_max_steps, seed=seed)
    model = MemoryPolicy(dtype=dtype, device=harness.dev, positions=updates * steps + 1)
    optimizer = torch.optim.Adam(model.parameters(), lr=1e-3)
    state = model.initial_state(actors)
    starts = torch.ones(actors, dtype=torch.bool, device=harness.dev)
    positions = torch.zeros(actors, dtype=torch.int32, device=harness.dev)
    rollout = Rollout(actors, steps, POOL[0] * POOL[1], harness.dev)
    losses, norms, episodes, apart, act_ms, learn_ms = [], [], 0, 0.0, [], []
    for _ in range(updates):
        torch.cuda.synchronize()
        began = time.perf_counter()
        collect(harness, model, rollout, state, starts, positions)
        torch.cuda.synchronize()
        collected = time.perf_counter()
        loss, norm, said = learn(model, optimizer, rollout, max_norm)
        torch.cuda.synchronize()
        act_ms.append((collected - began) * 1e3 / steps)
        learn_ms.append((time.perf_counter() - collected) * 1e3)
        losses.append(float(loss))
        norms.append(float(norm))
        episodes += int(rollout.starts[:, :-1].sum())
        apart = max(apart, float((said - rollout.acted).norm() / rollout.acted.norm()))
    return {"loss_first": losses[0], "loss_last": losses[-1], "grad_norm_first": norms[0], "grad_norm_last": norms[-1],
            "episodes": episodes, "acted_against_learned": apart,
            "act_ms": sorted(act_ms)[len(act_ms) // 2], "learn_ms": sorted(learn_ms)[len(learn_ms) // 2]}


def main(argv: list[str] | None = None) -> int:
    ap = argparse.ArgumentParser(description="Train a small memory policy on the tracer's observations (MI355X).")
    ap.add_argument("--gmdag-file", nargs="+", help="compiled .gmdag worlds (default: a seeded room with spheres)")
    ap.add_argument("--actors", type=int, default=64)
    ap.add_argument("--steps", type=int, default=128, help="frames of a rollout")
    ap.add_argument("--updates", type=int, default=10)
    ap.add_argument("--azimuth-bins", type=int, default=256)
    ap.add_argument("--elevation-bins", type=int, default=48)
    ap.add_argument("--max-distance", type=float, default=30.0)
    ap.add_argument("--sdf-max-steps", type=int, default=256)
    ap.add_argument("--seed", type=int, default=0)
    ap.add_argument("--json", action="store_true")
    args = ap.parse_args(argv)
    if min(args.actors, args.steps, args.updates) < 1:
        ap.error("actors, steps and updates must be >= 1")
    if args.gmdag_file:
        from .gmdag import load_gmdag_asset

        assets = [load_gmdag_asset(p) for p in args.gmdag_file]
        scenes = [(a.nodes, a.bbox_min, a.bbox_max) for a in assets]
    else:
        from . import scenes as S

        room = S.box_room()
        scenes = [(room.compile(), room.bbox_min, room.bbox_max)]
    summary = {"gmdag_file": [str(Path(f).expanduser()) for f in args.gmdag_file or []], "actors": args.actors,
               "steps": args.steps, "updates": args.updates,
               **run(scenes, actors=args.actors, steps=args.steps, updates=args.updates, azimuth_bins=args.azimuth_bins,
                     elevation_bins=args.elevation_bins, max_distance=args.max_distance,
                     sdf_max_steps=args.sdf_max_steps, seed=args.seed)}
    if args.json:
        print(json.dumps(summary, indent=2))
    else:
        print("memory-policy - " + ", ".join(f"{k}={v:.4g}" if isinstance(v, float) else f"{k}={v}"
                                             for k, v in summary.items() if k != "gmdag_file"))
    return 0


if __name__ == "__main__":
    sys.exit(main())

"""Definitions of a selective memory's operators in float64 on the CPU, token by token, for the tests
of ``navi_amd.policy``; gradients by autograd through them."""

from __future__ import annotations

import torch

from .policy_reference import ROUNDING


def rounding(t: torch.Tensor) -> float:
    """What rounding a tensor's numbers leaves of its 2-norm: half a step of each at most, and of many
    numbers (a thousand) the mean's share of that."""
    if t.dtype == torch.float32:
        return 0.0
    return ROUNDING[t.dtype] if t.numel() >= 1000 else torch.finfo(t.dtype).eps / 2


def scan(x, dt, a, b, c, d, dt_bias, starts, state):
    """(y, final state); ``a`` may be [Heads], or one rate for each token ([Envs, Steps, Heads])."""
    x, dt, a, b, c = (t.cpu().double() for t in (x, dt, a, b, c))
    envs, steps, heads, head_dim = x.shape
    share = heads // b.shape[2]
    s = torch.zeros(envs, heads, b.shape[3], head_dim, dtype=torch.float64) if state is None else state.cpu().double()
    z = dt if dt_bias is None else dt + dt_bias.cpu().double()
    beta = torch.clamp(z, min=0) + torch.log1p(torch.exp(-z.abs()))
    rates = a.expand(envs, steps, heads)
    out = []
    for t in range(steps):
        bt, ct = (u[:, t].repeat_interleave(share, dim=1) for u in (b, c))
        if starts is not None:
            s = torch.where(starts[:, t].cpu().bool()[:, None, None, None], torch.zeros_like(s), s)
        s = torch.exp(beta[:, t] * rates[:, t])[..., None, None] * s + (beta[:, t][..., None] * bt)[..., None] * x[:, t][..., None, :]
        y = (ct[..., None] * s).sum(-2)
        out.append(y if d is None else y + d.cpu().double()[:, None] * x[:, t])
    return torch.stack(out, 1) if out else x, s


def conv(x, weight, bias, starts, window, activation):
    """(y, window after)."""
    x, weight = x.cpu().double(), weight.cpu().double()
    envs, steps, channels = x.shape
    taps = weight.shape[1]
    held = [torch.zeros(envs, channels, dtype=torch.float64)] * (taps - 1)  # the latest last
    if window is not None:
        held = list(window.cpu().double().unbind(1))
    out = []
    for t in range(steps):
        if starts is not None:
            first = starts[:, t].cpu().bool()[:, None]
            held = [torch.where(first, torch.zeros_like(h), h) for h in held]
        taken = [*held, x[:, t]]
        z = sum(weight[:, k] * taken[k] for k in range(taps))
        z = z if bias is None else z + bias.cpu().double()
        out.append(z * torch.sigmoid(z) if activation == "silu" else z)
        held = taken[1:]
    return torch.stack(out, 1) if out else x, torch.stack(held, 1)


def block(y, residual, gate, scale, post, pre, eps, parts=False):
    """(stream, normed), with ``parts`` also the two norms before their weights."""
    y, residual = y.cpu().double(), residual.cpu().double()
    norm = lambda x: x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)  # noqa: E731
    m = first = norm(y)
    for factor in (post, None if gate is None else torch.sigmoid(gate.cpu().double()) * gate.cpu().double(), scale):
        m = m if factor is None else m * factor.cpu().double()
    h = residual + m
    second = norm(h)
    normed = second if pre is None else second * pre.cpu().double()
    return (h, normed, first, second) if parts else (h, normed)


def orthogonal(g, steps, factors, eps):
    a, b, c = factors
    x = g.detach().cpu().double()
    turned = x.shape[0] > x.shape[1]
    x = x.T if turned else x
    x = x / (x.norm() + eps)
    for _ in range(steps):
        gram = x @ x.T
        x = a * x + (b * gram + c * gram @ gram) @ x
    return x.T if turned else x

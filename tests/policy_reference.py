"""Definitions of the policy's operators in float64 on the CPU, token by token, for the tests
of ``navi_amd.policy``; gradients by autograd through them."""

from __future__ import annotations

import torch

EPS = 2.0 ** -24  # of float32, rounding to nearest
# the root mean square of a rounding's relative error, for bounds of 2-norms: 0.41 of the
# largest, 2^-8 for bfloat16 and 2^-11 for float16, rounded up to half of it
ROUNDING = {torch.float32: EPS, torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -12}


def rule(q, k, v, g, beta, starts, state, scale):
    """(o, final state): the recurrence in float64 on the CPU; ``starts`` and ``state`` may be None."""
    q, k, v, g, beta = (x.cpu().double() for x in (q, k, v, g, beta))
    envs, steps, heads, dim = v.shape
    share = heads // q.shape[2]
    s = torch.zeros(envs, heads, q.shape[3], dim, dtype=torch.float64) if state is None else state.cpu().double()
    out = []
    for t in range(steps):
        kt, qt = (x[:, t].repeat_interleave(share, dim=1) for x in (k, q))
        a = torch.exp(g[:, t])[..., None, None]
        if starts is not None:
            first = starts[:, t].cpu().bool()[:, None, None, None]
            s = torch.where(first, torch.zeros_like(s), s)
        s = torch.where(a == 0, torch.zeros_like(s), a * s)
        u = v[:, t] - (kt[..., None] * s).sum(-2)
        s = s + (beta[:, t][..., None] * kt)[..., None] * u[..., None, :]
        out.append(scale * (qt[..., None] * s).sum(-2))
    o = torch.stack(out, 1) if out else v
    return o, s


def norm(x, weight, cos, sin, positions, kind, eps, interleaved):
    """One of ``qk_norm``'s outputs in float64 on the CPU."""
    x = x.cpu().double()
    square = x.square().sum(-1, keepdim=True)
    y = x / torch.sqrt((square / x.shape[-1] if kind == "rms" else square) + eps)
    if weight is not None:
        y = y * weight.cpu().double()
    if cos is None:
        return y
    pairs = cos.shape[1]
    at = torch.arange(x.shape[1]).expand(x.shape[:2]) if positions is None else positions.cpu().long()
    c, s = (z.cpu().double()[at][:, :, None] for z in (cos, sin))
    if interleaved:
        a, b = y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = y[..., :pairs], y[..., pairs:2 * pairs]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([turned, y[..., 2 * pairs:]], -1)


def off(got, want) -> float:
    """The 2-norm of the difference over that of the wanted values."""
    got, want = got.detach().cpu().double(), want.detach()
    assert got.shape == want.shape
    assert torch.isfinite(got).all()
    size = float(want.norm())
    return float((got - want).norm()) / size if size else float((got - want).norm())

"""``qk_norm`` and ``clip_grad_norm`` (``navi_amd.policy``) on the GPU against float64.

Tolerances. A row's norm is a sum of squares in float32 whose relative error is a few 2^-24
whatever its length, and each output is a handful of products: 8 x 2^-24 of the norm, plus
the rounding of 16-bit outputs. Weight gradients add rows by the hundred
in float32, in groups: 32 x 2^-24.
"""

from __future__ import annotations

import math

import pytest
import torch

from . import policy_reference as ref

pytestmark = pytest.mark.gpu

TOL = 8 * ref.EPS


@pytest.fixture(scope="module")
def policy(gpu):
    from navi_amd import policy

    return policy


def tolerance(dtype):
    return TOL + (ref.ROUNDING[dtype] if dtype != torch.float32 else 0.0)


def tables(end, pairs, gen):
    angle = 6.3 * torch.rand(end, pairs, generator=gen)
    return torch.cos(angle).cuda(), torch.sin(angle).cuda()


CASES = [
    # envs, steps, query heads, key heads, dim, pairs, interleaved, kind, weights, dtype
    (1, 1, 1, 1, 1, 0, False, "rms", False, torch.float32),
    (2, 7, 4, 2, 64, 32, False, "rms", True, torch.bfloat16),
    (2, 7, 4, 2, 64, 16, False, "l2", False, torch.float16),
    (3, 5, 3, 1, 128, 64, True, "rms", True, torch.float32),
    (3, 5, 3, 1, 40, 10, False, "rms", True, torch.float32),
    (3, 5, 2, 2, 33, 16, True, "l2", True, torch.bfloat16),
    (2, 3, 1, 1, 96, 24, False, "rms", False, torch.float32),
    (2, 9, 2, 1, 256, 128, False, "rms", True, torch.bfloat16),
    (1, 4, 1, 1, 512, 256, False, "rms", True, torch.float32),
    (1, 4, 2, 1, 1000, 333, True, "l2", True, torch.float32),
    (16, 130, 4, 4, 64, 32, False, "l2", True, torch.bfloat16),
]


@pytest.mark.parametrize("given", [True, False], ids=["positions", "steps"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_norm_and_gradients(policy, case, given):
    envs, steps, hq, hk, dim, pairs, interleaved, kind, weights, dtype = case
    gen = torch.Generator().manual_seed(dim)
    x = {"q": torch.randn(envs, steps, hq, dim, generator=gen).to(dtype).cuda(),
         "k": (5 * torch.randn(envs, steps, hk, dim, generator=gen)).to(dtype).cuda()}
    w = {n: (1 + 0.3 * torch.randn(dim, generator=gen)).cuda() if weights else None for n in x}
    cos = sin = positions = None
    if pairs:
        cos, sin = tables(steps + 30, pairs, gen)
        if given:
            positions = torch.randint(0, steps + 30, (envs, steps), generator=gen).to(
                torch.int64 if dim % 2 else torch.int32).cuda()
    leaves = {n: t.clone().requires_grad_() for n, t in x.items()}
    scales = {n: t.clone().requires_grad_() if weights else None for n, t in w.items()}
    got = policy.qk_norm(leaves["q"], leaves["k"], q_weight=scales["q"], k_weight=scales["k"], norm=kind, eps=1e-5,
                         cos=cos, sin=sin, positions=positions, interleaved=interleaved)
    for n, y in zip(x, got):
        exact = x[n].cpu().double().requires_grad_()
        scale = w[n].cpu().double().requires_grad_() if weights else None
        want = ref.norm(exact, scale, cos, sin, positions, kind, 1e-5, interleaved)
        assert y.dtype == dtype and y.is_contiguous()
        assert ref.off(y, want) <= tolerance(dtype)
        grad = torch.randn(y.shape, generator=gen).to(dtype)
        wanted = torch.autograd.grad(want, [exact] + ([scale] if weights else []), grad.double())
        back = torch.autograd.grad(y, [leaves[n]] + ([scales[n]] if weights else []), grad.cuda(), retain_graph=True)
        # dx is the part of a row across x: its norm may be smaller than what it is made of
        room = tolerance(dtype) * float(wanted[0].norm()) + 4 * TOL * float((wanted[0].norm() if dim > 1 else grad.double().norm()))
        assert float((back[0].cpu().double() - wanted[0]).norm()) <= room
        if weights:
            assert ref.off(back[1], wanted[1]) <= 32 * ref.EPS


def test_rows_of_zeros_and_of_large_numbers(policy):
    q = torch.zeros(1, 2, 1, 64, device="cuda")
    q[0, 1] = 1e15
    k = torch.full_like(q, 1e-15)
    a, b = policy.qk_norm(q, k, norm="rms", eps=1e-6)
    assert torch.equal(a[0, 0], torch.zeros_like(a[0, 0]))
    assert torch.allclose(a[0, 1], torch.ones_like(a[0, 1]))
    assert torch.allclose(b, torch.full_like(b, 1e-12), rtol=1e-6, atol=0.0)


def test_positions_outside_the_tables(policy):
    q = torch.randn(2, 3, 2, 64, device="cuda")
    cos, sin = torch.ones(4, 16, device="cuda"), torch.zeros(4, 16, device="cuda")
    positions = torch.tensor([[0, 4, 1], [3, -1, 2]], device="cuda")
    for interleaved in (False, True):
        a, _ = policy.qk_norm(q, q, cos=cos, sin=sin, positions=positions, interleaved=interleaved)
        bad = torch.isnan(a[..., :32]).all(-1).all(-1)
        assert torch.equal(bad, (positions < 0) | (positions >= 4))
        assert torch.isfinite(a[..., 32:]).all()


def test_views_and_odd_addresses(policy):
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(2, 9, 6 * 64 + 1, generator=gen, device="cuda").bfloat16()
    cos, sin = torch.rand(9, 32, generator=gen, device="cuda"), torch.rand(9, 32, generator=gen, device="cuda")
    for first in (0, 1):
        part = x[..., first:first + 384].unflatten(-1, (6, 64))
        q, k = part[:, :, :4], part[:, :, 4:]
        q1, k1 = (t.detach().requires_grad_() for t in (q, k))
        q2, k2 = (t.contiguous().detach().requires_grad_() for t in (q, k))
        got = policy.qk_norm(q1, k1, cos=cos, sin=sin)
        want = policy.qk_norm(q2, k2, cos=cos, sin=sin)
        for a, b in zip(got, want):
            assert float((a - b).abs().max()) <= 2.0 ** -7 * float(b.abs().max())  # (one unit: another order of sums)
        back = torch.autograd.grad([got[0].float().sum() + got[1].float().sum()], [q1, k1])
        same = torch.autograd.grad([want[0].float().sum() + want[1].float().sum()], [q2, k2])
        for a, b in zip(back, same):
            assert float((a - b).float().norm()) <= 2.0 ** -7 * float(b.float().norm())


def test_norm_of_nothing(policy):
    q, k = torch.zeros(2, 0, 3, 64, device="cuda"), torch.zeros(2, 0, 1, 64, device="cuda")
    w = torch.ones(64, device="cuda", requires_grad=True)
    a, b = policy.qk_norm(q, k, q_weight=w, k_weight=w)
    assert a.shape == q.shape and b.shape == k.shape
    assert torch.equal(torch.autograd.grad(a.sum() + b.sum(), w)[0], torch.zeros(64, device="cuda"))


def test_norm_refusals(policy):
    q, k = torch.zeros(2, 3, 4, 64, device="cuda"), torch.zeros(2, 3, 2, 64, device="cuda")
    cos = torch.zeros(5, 32, device="cuda")
    bad = [
        (dict(q=q.cpu()), "q must be a CUDA tensor"),
        (dict(k=k.half()), "k must be float32"),
        (dict(k=k[:, :2]), "q and k must be"),
        (dict(k=k[..., :32]), "q and k must be"),
        (dict(norm="max"), "norm must be"),
        (dict(eps=-1.0), "eps must be"),
        (dict(q_weight=torch.zeros(32, device="cuda")), "q_weight must be"),
        (dict(k_weight=torch.zeros(64, device="cuda").half()), "k_weight must be float32"),
        (dict(cos=cos), "cos and sin go together"),
        (dict(cos=cos, sin=cos[:, :8]), "cos and sin must be alike"),
        (dict(cos=torch.zeros(5, 33, device="cuda"), sin=torch.zeros(5, 33, device="cuda")), "cos and sin must be"),
        (dict(positions=torch.zeros(2, 3, dtype=torch.int32, device="cuda")), "positions need"),
        (dict(cos=cos, sin=cos, positions=torch.zeros(2, 3, device="cuda")), "positions must be int32 or int64"),
        (dict(cos=cos, sin=cos, positions=torch.zeros(3, 2, dtype=torch.int32, device="cuda")), "positions must be"),
        (dict(q=q.transpose(2, 3)), "q and k must be"),
    ]
    for over, words in bad:
        with pytest.raises(RuntimeError, match=words):
            policy.qk_norm(over.pop("q", q), over.pop("k", k), **over)


# ---- clipping ----


def shapes(n):
    return [((3 + 7 * i) % 50 + 1, (5 + 3 * i) % 90 + 1) for i in range(n)]


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("max_norm", [0.5, 1e6, 0.0])
@pytest.mark.parametrize("count", [1, 5, 111, 112, 113, 400])
def test_clip(policy, count, max_norm, in_place):
    gen = torch.Generator().manual_seed(count)
    kinds = (torch.float32, torch.bfloat16, torch.float16)
    grads = [torch.randn(s, generator=gen).to(kinds[i % 3]).cuda() for i, s in enumerate(shapes(count))]
    before = [g.clone() for g in grads]
    out = None if in_place else [torch.full_like(g, 7.0) for g in grads]
    norm = policy.clip_grad_norm(grads, max_norm, out=out)
    want = math.sqrt(sum(float(g.double().square().sum()) for g in before))
    assert norm.dim() == 0 and norm.dtype == torch.float32
    assert abs(float(norm) - want) <= 4 * ref.EPS * want
    factor = torch.clamp(max_norm / (norm.cpu() + 1e-6), max=1.0)  # (in float32, as the kernel's)
    for g, b, o in zip(grads, before, grads if in_place else out):
        assert in_place or torch.equal(g, b)
        assert torch.equal(o.cpu(), (b.cpu().float() * factor).to(o.dtype))  # one product, rounded once


def test_clip_lengths_and_addresses(policy):
    """Every length and start within a vector, guards on both sides."""
    for dtype in (torch.float32, torch.bfloat16):
        flat = torch.randn(4000, device="cuda").to(dtype)
        kept = flat.clone()
        out = torch.full_like(flat, 3.0)
        spans = [(1 + 40 * i + i % 9, 1 + i % 17) for i in range(90)]
        norm = policy.clip_grad_norm([flat[a:a + n] for a, n in spans], 0.25, out=[out[a:a + n] for a, n in spans])
        inside = torch.zeros(4000, dtype=torch.bool, device="cuda")
        for a, n in spans:
            inside[a:a + n] = True
        want = float(kept[inside].double().norm())
        assert abs(float(norm) - want) <= 4 * ref.EPS * want
        assert torch.equal(flat, kept)
        assert torch.equal(out[~inside], torch.full_like(out[~inside], 3.0))
        assert torch.allclose(out[inside].double(), kept[inside].double() * 0.25 / want, rtol=2 * ref.ROUNDING[dtype] + 1e-6, atol=0)


def test_clip_large_tensors_and_orders(policy):
    a = torch.randn(513, 4099, device="cuda")
    b = torch.randn(300, 70, 11, device="cuda").permute(2, 0, 1)  # dense, not contiguous
    want = math.sqrt(float(a.double().square().sum() + b.double().square().sum()))
    clean = [a.clone(), b.clone()]
    norm = policy.clip_grad_norm([a, None, b, torch.empty(0, device="cuda")], 1.0)
    assert abs(float(norm) - want) <= 4 * ref.EPS * want
    for x, y in zip((a, b), clean):
        assert torch.allclose(x.double(), y.double() / (want + 1e-6), rtol=TOL, atol=0)


def test_clip_of_numbers_that_are_not_finite(policy):
    for bad, rest in ((math.nan, math.nan), (math.inf, 0.0)):
        g = torch.ones(1000, device="cuda")
        h = torch.ones(10, device="cuda")
        g[500] = bad
        norm = policy.clip_grad_norm([g, h], 1.0)
        assert math.isnan(float(norm)) if math.isnan(bad) else float(norm) == math.inf
        assert math.isnan(float(g[500]))
        assert torch.equal(torch.nan_to_num(h, nan=-1.0), torch.full_like(h, -1.0 if math.isnan(rest) else 0.0))


def test_clip_gives_the_same_bits(policy):
    grads = [torch.randn(s, device="cuda") for s in shapes(200)] + [torch.randn(1 << 22, device="cuda")]
    out = [torch.empty_like(g) for g in grads]
    first = policy.clip_grad_norm(grads, 1.0, out=out)
    kept = [o.clone() for o in out]
    for _ in range(3):
        assert torch.equal(policy.clip_grad_norm(grads, 1.0, out=out), first)
        assert all(torch.equal(a, b) for a, b in zip(out, kept))


def test_clip_refusals(policy):
    g = torch.ones(4, 4, device="cuda")
    bad = [
        (([], 1.0), {}, "at least one"),
        (([None], 1.0), {}, "at least one"),
        (([g.cpu()], 1.0), {}, "CUDA"),
        (([g.double()], 1.0), {}, "float32, bfloat16 or float16"),
        (([g[:, :2]], 1.0), {}, "without gaps"),
        (([g], -1.0), {}, "not be negative"),
        (([g], math.nan), {}, "not be negative"),
        (([g], 1.0), {"out": []}, "as long as"),
        (([g], 1.0), {"out": [g.half()]}, "out must be like"),
        (([g], 1.0), {"out": [torch.ones(4, 8, device="cuda")[:, ::2]]}, "out must be like"),
    ]
    for args, more, words in bad:
        with pytest.raises(RuntimeError, match=words):
            policy.clip_grad_norm(*args, **more)

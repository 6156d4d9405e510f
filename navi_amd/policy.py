"""Operators of a policy with a memory, over the tracer's observations, and of its training step.

The reference's policies are PyTorch modules (``projects/actor``: an encoder of the
``(B, 3, Az, El)`` observation, a temporal core, PPO heads) around the in-process tracer.
These are the operators of such a core as HIP kernels:

* ``gated_delta_rule`` / ``gated_delta_step``: a memory of one ``K x V`` matrix ``S`` per
  head that writes by error correction. With ``a = 0`` at the first token of an episode and
  ``exp(g)`` elsewhere: ``u = v - a S^T k``, ``S <- a S + beta k u^T``, ``o = scale S^T q``.
  One takes whole rollouts in chunks of 64 tokens, with gradients, the other a frame of every
  environment; both give the same outputs.
* ``qk_norm``: norms of queries and keys for each head and the rotation by position.
* ``clip_grad_norm``: the norm of all gradients, and their clipping by it.

The kernels run on PyTorch's current stream, never wait for the device and keep nothing of a
call; queries, keys and values may be views of one projection (any strides but the last
axis's). Misuse raises ``RuntimeError``; there is no CPU fallback.
"""

from __future__ import annotations

import ctypes
import math
from typing import Iterable

import torch
from torch.autograd.function import once_differentiable

from . import _policy_native as _native

__all__ = ["gated_delta_rule", "gated_delta_step", "qk_norm", "clip_grad_norm"]

_DTYPES = {torch.float32: _native.F32, torch.bfloat16: _native.BF16, torch.float16: _native.F16}
_MASKS = (torch.bool, torch.uint8)


def _check(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def _check_tensor(name: str, t, dtypes, dims: int, device=None) -> None:
    _check(isinstance(t, torch.Tensor) and t.is_cuda, f"{name} must be a CUDA tensor")
    _check(t.dtype in dtypes, f"{name} must be {' or '.join(str(d).replace('torch.', '') for d in dtypes)}")
    _check(t.dim() == dims, f"{name} must have {dims} dimensions")
    _check(device is None or t.device == device, f"{name} must be on the same device as q ({device})")


def _dense_last(t: torch.Tensor) -> bool:
    return t.stride(-1) == 1 or t.size(-1) <= 1


def _stream(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


def _written(t: torch.Tensor) -> None:
    """Tells autograd of a write by a kernel."""
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


# ---- the gated delta rule ----


def _check_rule(q, k, v, g, beta, starts, lead: tuple[str, ...]) -> None:
    n = len(lead)
    shape = ", ".join(lead)
    _check_tensor("q", q, tuple(_DTYPES), n + 2)
    for name, t in (("k", k), ("v", v)):
        _check_tensor(name, t, (q.dtype,), n + 2, q.device)
    for name, t in (("g", g), ("beta", beta)):
        _check_tensor(name, t, (torch.float32,), n + 1, q.device)
    for name, t in (("q", q), ("k", k), ("v", v)):
        _check(_dense_last(t), f"{name} must be contiguous in its last dimension")
    _check(q.shape == k.shape, f"q and k must both be [{shape}, KeyHeads, KeyDim]")
    _check(v.shape[:n] == q.shape[:n], f"v must be [{shape}, ValueHeads, ValueDim] like q")
    hk, hv = q.size(n), v.size(n)
    _check(hk > 0 and hv > 0 and hv % hk == 0, "the value heads must be a multiple of the key heads")
    _check(0 < q.size(-1) <= _native.MAX_KEY_DIM, f"the key dimension must be in [1, {_native.MAX_KEY_DIM}]")
    _check(v.size(-1) > 0, "the value dimension must be positive")
    for name, t in (("g", g), ("beta", beta)):
        _check(t.shape == v.shape[:-1], f"{name} must be [{shape}, ValueHeads]")
    if starts is not None:
        _check_tensor("starts", starts, _MASKS, n, q.device)
        _check(starts.shape == q.shape[:n], f"starts must be [{shape}]")


def _check_state(name: str, state, q, v, envs: int) -> None:
    _check_tensor(name, state, (torch.float32,), 4, q.device)
    want = (envs, v.size(-2), q.size(-1), v.size(-1))
    _check(tuple(state.shape) == want, f"{name} must be [Envs, ValueHeads, KeyDim, ValueDim] = {list(want)}")
    _check(state.is_contiguous(), f"{name} must be contiguous")


_FARTHEST = ((1 << 31) - 1) // _native.CHUNK - (1 << 18)  # bytes between steps that the chunked kernels reach


def _rows_apart(t: torch.Tensor) -> torch.Tensor:
    """``t`` as the chunked kernels read it: steps that do not overlap (an expanded axis) and lie
    within reach; else a copy."""
    if t.size(1) <= 1 or t.size(3) <= t.stride(1) <= _FARTHEST // t.element_size():
        return t
    return t.contiguous()


def _strides(t: torch.Tensor, step: bool) -> ctypes.Array:
    s = t.stride()
    return (ctypes.c_int64 * 3)(s[0], s[1], s[2]) if step else (ctypes.c_int64 * 3)(s[0], 0, s[1])


def _rule_args(q, k, v, g, beta, starts, scale, initial_state, out, final_state, step=True) -> _native.DeltaRule:
    a = _native.DeltaRule(
        dtype=_DTYPES[q.dtype], key_heads=q.size(-2), value_heads=v.size(-2), key_dim=q.size(-1),
        value_dim=v.size(-1), envs=q.size(0), steps=q.size(1) if step else 1, scale=scale, q=q.data_ptr(),
        k=k.data_ptr(), v=v.data_ptr(), q_stride=_strides(q, step), k_stride=_strides(k, step),
        v_stride=_strides(v, step), g=g.data_ptr(), beta=beta.data_ptr(), g_stride=_strides(g, step),
        beta_stride=_strides(beta, step), initial_state=_ptr(initial_state), out=_ptr(out),
        final_state=_ptr(final_state))
    if starts is not None:
        a.starts = starts.data_ptr()
        a.starts_stride = (ctypes.c_int64 * 2)(starts.stride(0), starts.stride(1) if step else 0)
    return a


def _forward(q, k, v, g, beta, starts, scale, initial_state, return_state, save):
    """(out, final state or None, matrices, states, updates): the last three for a backward pass."""
    envs, steps, heads, dim = v.shape
    out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    state = states = updates = None
    if return_state:
        state = torch.empty((envs, heads, q.size(-1), dim), dtype=torch.float32, device=v.device)
    chunks = -(-steps // _native.CHUNK)
    matrices = torch.empty((envs * heads, chunks, _native.CHUNK_MATRICES), dtype=torch.float32, device=v.device)
    if save:
        states = torch.empty((envs * heads, max(0, chunks - 1), q.size(-1), dim), dtype=torch.float32, device=v.device)
        updates = torch.empty((envs * heads, steps, dim), dtype=torch.float32, device=v.device)
    a = _rule_args(q, k, v, g, beta, starts, scale, initial_state, out, state)
    a.matrices, a.states, a.updates = matrices.data_ptr(), _ptr(states), _ptr(updates)
    scratch = _native.check(_native.lib().navi_delta_scratch(ctypes.byref(a)))
    if scratch:
        scratch = torch.empty(scratch // 4, dtype=torch.float32, device=v.device)
        a.scratch = scratch.data_ptr()
    with torch.cuda.device(q.device):
        _native.check(_native.lib().navi_delta_forward(ctypes.byref(a), _stream(q.device)))
    return out, state, matrices, states, updates


class _DeltaRule(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, initial_state, starts, scale, return_state):
        out, state, *saved = _forward(q, k, v, g, beta, starts, scale, initial_state, return_state, True)
        ctx.save_for_backward(q, k, v, g, beta, initial_state, starts, *saved)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return (out, state) if return_state else out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out, grad_state=None):
        q, k, v, g, beta, initial_state, starts, matrices, states, updates = ctx.saved_tensors
        if grad_out is None and grad_state is None:
            return (None,) * 9
        if grad_out is None:
            grad_out = torch.zeros((), dtype=v.dtype, device=v.device).expand(v.shape)
        if not _dense_last(grad_out):  # (of a broadcast, for one)
            grad_out = grad_out.contiguous()
        grad_out = _rows_apart(grad_out)
        if grad_state is not None:
            grad_state = grad_state.contiguous()
        d_q, d_k, d_v, d_g, d_beta = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v, g, beta))
        d_state = torch.empty_like(initial_state) if initial_state is not None and ctx.needs_input_grad[5] else None
        if v.numel() == 0:
            if d_state is not None:
                d_state = torch.zeros_like(d_state) if grad_state is None else grad_state.clone()
            return d_q, d_k, d_v, d_g, d_beta, d_state, None, None, None
        a = _rule_args(q, k, v, g, beta, starts, ctx.scale, initial_state, grad_out, None)
        a.matrices, a.states, a.updates = matrices.data_ptr(), states.data_ptr(), updates.data_ptr()
        lib = _native.lib()
        size = _native.check(lib.navi_delta_workspace(ctypes.byref(a)))
        workspace = torch.empty(size // 4, dtype=torch.float32, device=q.device)
        d = _native.DeltaGradients(
            grad_out=grad_out.data_ptr(), grad_out_stride=_strides(grad_out, True), grad_final_state=_ptr(grad_state),
            d_q=d_q.data_ptr(), d_k=d_k.data_ptr(), d_v=d_v.data_ptr(), d_g=d_g.data_ptr(), d_beta=d_beta.data_ptr(),
            d_initial_state=_ptr(d_state), workspace=workspace.data_ptr())
        with torch.cuda.device(q.device):
            _native.check(lib.navi_delta_backward(ctypes.byref(a), ctypes.byref(d), _stream(q.device)))
        return d_q, d_k, d_v, d_g, d_beta, d_state, None, None, None


def gated_delta_rule(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor, *,
                     scale: float | None = None, starts: torch.Tensor | None = None,
                     initial_state: torch.Tensor | None = None, return_state: bool = False):
    """The gated delta rule over whole rollouts, differentiable in q, k, v, g, beta and
    initial_state.

    ``q``, ``k``: ``[Envs, Steps, KeyHeads, KeyDim]`` in float32, bfloat16 or float16 (key
    dimension up to 128), ``v``: ``[Envs, Steps, ValueHeads, ValueDim]`` of the same type, with
    ``ValueHeads`` a multiple of ``KeyHeads`` (value head h reads key head
    ``h // (ValueHeads // KeyHeads)``). ``g`` (the logarithm of the decay, at most 0; -inf
    forgets everything) and ``beta``: ``[Envs, Steps, ValueHeads]`` float32. ``starts``:
    ``[Envs, Steps]`` bool or uint8, tokens that begin an episode: the state before one is
    forgotten (at the first step, whatever it holds). ``initial_state``: ``[Envs, ValueHeads, KeyDim, ValueDim]``
    float32, zeros by default. ``scale`` defaults to ``KeyDim ** -0.5``.

    Returns ``o`` like ``v``, with ``return_state`` also the state after the last token. Keys
    are meant to have norm 1 (``qk_norm`` with ``norm="l2"``) and beta to lie in [0, 1]: the
    memory contracts then. Arithmetic is of float32's precision for every type, rounded
    once at the end. A NaN or infinity in the inputs may reach every token of its chunk of 64
    tokens and what follows them, beyond the start of an episode too.
    """
    _check_rule(q, k, v, g, beta, starts, ("Envs", "Steps"))
    if initial_state is not None:
        _check_state("initial_state", initial_state, q, v, q.size(0))
    scale = q.size(-1) ** -0.5 if scale is None else float(scale)
    q, k, v = (_rows_apart(t) for t in (q, k, v))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, g, beta, initial_state)):
        return _DeltaRule.apply(q, k, v, g, beta, initial_state, starts, scale, bool(return_state))
    out, state, *_ = _forward(q, k, v, g, beta, starts, scale, initial_state, return_state, False)
    return (out, state) if return_state else out


def gated_delta_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                     state: torch.Tensor, *, scale: float | None = None, starts: torch.Tensor | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """One token of every environment: ``gated_delta_rule`` without the ``Steps`` axis.

    ``state`` (float32, ``[Envs, ValueHeads, KeyDim, ValueDim]``) is updated in place; the
    output goes to ``out`` (like ``v``, contiguous) if given. No gradients: this is the form
    for acting.
    """
    _check_rule(q, k, v, g, beta, starts, ("Envs",))
    _check_state("state", state, q, v, q.size(0))
    _check(not (torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, g, beta, state))),
           "gated_delta_step has no gradients; use gated_delta_rule, or torch.no_grad()")
    if out is None:
        out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    else:
        _check_tensor("out", out, (v.dtype,), 3, q.device)
        _check(out.shape == v.shape and out.is_contiguous(), "out must be like v, contiguous")
    a = _rule_args(q, k, v, g, beta, starts, q.size(-1) ** -0.5 if scale is None else float(scale), state, out, state,
                   step=False)
    with torch.cuda.device(q.device):
        _native.check(_native.lib().navi_delta_step(ctypes.byref(a), _stream(q.device)))
    _written(state)
    return out


# ---- norms of queries and keys, rotation by position ----


def _norm_args(q, k, q_weight, k_weight, cos, sin, positions, norm, eps, interleaved) -> _native.QkNorm:
    a = _native.QkNorm(
        dtype=_DTYPES[q.dtype], norm=_NORMS[norm], query_heads=q.size(2), key_heads=k.size(2), head_dim=q.size(3),
        pairs=0 if cos is None else cos.size(1), interleaved=int(interleaved), envs=q.size(0), steps=q.size(1),
        eps=eps, q=q.data_ptr(), k=k.data_ptr(), q_stride=_strides(q, True), k_stride=_strides(k, True),
        q_weight=_ptr(q_weight), k_weight=_ptr(k_weight), cos=_ptr(cos), sin=_ptr(sin),
        positions_end=0 if cos is None else cos.size(0))
    if positions is not None:
        a.positions = positions.data_ptr()
        a.positions_stride = (ctypes.c_int64 * 2)(*positions.stride())
        a.positions_wide = int(positions.dtype == torch.int64)
    return a


_NORMS = {"rms": _native.NORM_RMS, "l2": _native.NORM_L2}


class _QkNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, norm, eps, interleaved):
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.rest = (norm, eps, interleaved)
        ctx.set_materialize_grads(False)
        return _norm_forward(q, k, q_weight, k_weight, cos, sin, positions, norm, eps, interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_q, grad_k):
        q, k, q_weight, k_weight, cos, sin, positions = ctx.saved_tensors
        if grad_q is None and grad_k is None:
            return (None,) * 10
        grads = []
        for grad, t in ((grad_q, q), (grad_k, k)):
            if grad is None:
                grad = torch.zeros((), dtype=t.dtype, device=t.device).expand(t.shape)
            grads.append(grad if _dense_last(grad) else grad.contiguous())
        grad_q, grad_k = grads
        a = _norm_args(q, k, q_weight, k_weight, cos, sin, positions, *ctx.rest)
        d_q, d_k = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k))
        weights = [torch.empty_like(w) if w is not None and ctx.needs_input_grad[2 + i] else None
                   for i, w in enumerate((q_weight, k_weight))]
        a.grad_q, a.grad_k, a.d_q, a.d_k = grad_q.data_ptr(), grad_k.data_ptr(), d_q.data_ptr(), d_k.data_ptr()
        a.grad_q_stride, a.grad_k_stride = _strides(grad_q, True), _strides(grad_k, True)
        a.d_q_weight, a.d_k_weight = _ptr(weights[0]), _ptr(weights[1])
        lib = _native.lib()
        if any(w is not None for w in weights):
            size = _native.check(lib.navi_qk_norm_workspace(ctypes.byref(a)))
            partial = torch.empty(size // 4, dtype=torch.float32, device=q.device)
            a.partial = partial.data_ptr()
        with torch.cuda.device(q.device):
            _native.check(lib.navi_qk_norm_backward(ctypes.byref(a), _stream(q.device)))
        return d_q, d_k, weights[0], weights[1], None, None, None, None, None, None


def _norm_forward(q, k, q_weight, k_weight, cos, sin, positions, norm, eps, interleaved):
    a = _norm_args(q, k, q_weight, k_weight, cos, sin, positions, norm, eps, interleaved)
    q_out, k_out = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k))
    a.q_out, a.k_out = q_out.data_ptr(), k_out.data_ptr()
    with torch.cuda.device(q.device):
        _native.check(_native.lib().navi_qk_norm(ctypes.byref(a), _stream(q.device)))
    return q_out, k_out


def qk_norm(q: torch.Tensor, k: torch.Tensor, *, q_weight: torch.Tensor | None = None,
            k_weight: torch.Tensor | None = None, norm: str = "rms", eps: float = 1e-6,
            cos: torch.Tensor | None = None, sin: torch.Tensor | None = None,
            positions: torch.Tensor | None = None, interleaved: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """Norms of queries and keys for each head, and the rotation by position in the same pass;
    differentiable in q, k and the weights.

    ``q``: ``[Envs, Steps, QueryHeads, HeadDim]`` and ``k``: ``[Envs, Steps, KeyHeads, HeadDim]``
    in float32, bfloat16 or float16 (head dimension up to 1024). ``norm="rms"`` divides by the
    root of the mean square plus eps, ``"l2"`` by that of the sum (rows of norm 1, what the
    gated delta rule takes). ``q_weight``, ``k_weight``: float32 ``[HeadDim]`` factors.
    ``cos``, ``sin``: float32 ``[Positions, Pairs]`` tables that rotate the first ``2 * Pairs``
    numbers of a row, pair i being (i, i + Pairs), or (2 i, 2 i + 1) with ``interleaved``.
    ``positions``: ``[Envs, Steps]`` int32 or int64 rows of the tables (a token's step by
    default); one outside the tables gives NaN in the numbers that it would rotate.
    """
    _check_tensor("q", q, tuple(_DTYPES), 4)
    _check_tensor("k", k, (q.dtype,), 4, q.device)
    _check(q.shape[:2] == k.shape[:2] and q.size(3) == k.size(3), "q and k must be [Envs, Steps, Heads, HeadDim], alike but for Heads")
    _check(0 < q.size(3) <= _native.MAX_NORM_DIM, f"the head dimension must be in [1, {_native.MAX_NORM_DIM}]")
    _check(_dense_last(q) and _dense_last(k), "q and k must be contiguous in their last dimension")
    _check(norm in _NORMS, "norm must be 'rms' or 'l2'")
    eps = float(eps)
    _check(math.isfinite(eps) and eps >= 0.0, "eps must be finite and not negative")
    for name, t in (("q_weight", q_weight), ("k_weight", k_weight)):
        if t is not None:
            _check_tensor(name, t, (torch.float32,), 1, q.device)
            _check(t.size(0) == q.size(3) and t.is_contiguous(), f"{name} must be [HeadDim], contiguous")
    _check((cos is None) == (sin is None), "cos and sin go together")
    if cos is not None:
        for name, t in (("cos", cos), ("sin", sin)):
            _check_tensor(name, t, (torch.float32,), 2, q.device)
            _check(t.shape == cos.shape and t.is_contiguous(), "cos and sin must be alike and contiguous")
        _check(cos.size(0) > 0 and 0 < 2 * cos.size(1) <= q.size(3), "cos and sin must be [Positions, Pairs], 2 * Pairs <= HeadDim")
    if positions is not None:
        _check(cos is not None, "positions need cos and sin")
        _check_tensor("positions", positions, (torch.int32, torch.int64), 2, q.device)
        _check(positions.shape == q.shape[:2], "positions must be [Envs, Steps]")
    args = (q, k, q_weight, k_weight, cos, sin, positions, norm, eps, bool(interleaved))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args[:4]):
        return _QkNorm.apply(*args)
    return _norm_forward(*args)


# ---- the norm of all gradients ----


def clip_grad_norm(grads: Iterable[torch.Tensor | None], max_norm: float, *, eps: float = 1e-6,
                   out: Iterable[torch.Tensor | None] | None = None) -> torch.Tensor:
    """Scales gradients by ``min(1, max_norm / (norm + eps))``, ``norm`` the root of the sum of
    all their squares, and returns ``norm`` (a float32 scalar on the device; nothing waits).

    ``grads``: float32, bfloat16 and float16 tensors of one device in any mix (None is
    skipped); each must fill its memory without gaps, in any order of its axes. They are
    scaled in place, or into ``out``, tensors of the same shapes, types and strides (views of
    an optimizer's flat buffer, for one). A norm that is not finite spoils the gradients as
    the formula says: NaN gives NaN, infinity gives 0 (NaN where the gradient is infinite).
    """
    max_norm, eps = float(max_norm), float(eps)
    _check(max_norm >= 0.0 and eps >= 0.0, "max_norm and eps must not be negative")
    grads = list(grads)
    to = grads if out is None else list(out)
    _check(len(to) == len(grads), "out must be as long as grads")
    pairs = [(x, y) for x, y in zip(grads, to) if x is not None]
    _check(len(pairs) > 0, "grads must hold at least one tensor")
    device = pairs[0][0].device
    for x, y in pairs:
        _check(isinstance(x, torch.Tensor) and x.is_cuda and x.layout == torch.strided, "grads must be dense CUDA tensors")
        _check(x.dtype in _DTYPES, "grads must be float32, bfloat16 or float16")
        _check(x.device == device, "grads must be on one device")
        _check(x.is_contiguous() or torch.ops.aten.is_non_overlapping_and_dense(x), "grads must fill their memory without gaps")
        if y is not x:
            _check(isinstance(y, torch.Tensor) and y.dtype == x.dtype and y.shape == x.shape and y.device == device
                   and (y.is_contiguous() if x.is_contiguous() else y.stride() == x.stride()),
                   "out must be like grads in shapes, types, strides and device")
    n = len(pairs)
    norm = torch.empty((), dtype=torch.float32, device=device)
    partial = torch.empty(_native.NORM_PARTIALS, dtype=torch.float32, device=device)
    with torch.cuda.device(device):
        _native.check(_native.lib().navi_clip_grad_norm(
            n, (ctypes.c_void_p * n)(*[x.data_ptr() for x, _ in pairs]),
            (ctypes.c_void_p * n)(*[y.data_ptr() for _, y in pairs]),
            (ctypes.c_int64 * n)(*[x.numel() for x, _ in pairs]),
            (ctypes.c_int32 * n)(*[_DTYPES[x.dtype] for x, _ in pairs]),
            max_norm, eps, norm.data_ptr(), partial.data_ptr(), _stream(device)))
    for _, y in pairs:
        _written(y)
    return norm

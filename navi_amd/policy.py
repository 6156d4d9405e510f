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
axis's). Misuse raises ``RuntimeError``, forward-mode derivatives do too; there is no CPU fallback.
"""

from __future__ import annotations

import math
import struct
from typing import Iterable

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _policy_native as _native

__all__ = ["gated_delta_rule", "gated_delta_step", "qk_norm", "clip_grad_norm"]

_DTYPES = {torch.float32: _native.F32, torch.bfloat16: _native.BF16, torch.float16: _native.F16}
_MASKS = (torch.bool, torch.uint8)

# Arguments are looked over twice: `_fine` in one expression on every call (a call of one frame
# is bound by the host), and by name, for the message, where that found something.


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


def _check_tangents(*tensors) -> None:
    """The kernels would drop the tangents of forward-mode derivatives without a word."""
    if forward_ad._current_level >= 0:  # (within a dual_level only)
        _check(all(t is None or forward_ad.unpack_dual(t).tangent is None for t in tensors),
               "the policy's operators have no forward-mode derivatives")


def _call(function, device: torch.device, *args) -> None:
    """An entry point on the device's current stream."""
    index = device.index
    if index == torch.cuda.current_device():
        code = function(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            code = function(*args, torch._C._cuda_getCurrentRawStream(index))
    if code:
        _native.check(code)


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _written(tensors: list[torch.Tensor]) -> None:
    """Tells autograd of writes by a kernel."""
    tensors = [t for t in tensors if not t.is_inference()]
    if tensors:
        torch.autograd.graph.increment_version(tensors)


# ---- the gated delta rule ----


def _fine_rule(q, k, v, g, beta, starts) -> bool:
    """Whether the inputs are in order ([Envs, Steps, ...] and [Envs, ...] alike)."""
    try:
        lead, device, dtype = q.shape[:-2], q.device, q.dtype
        (hk, kd), (hv, vd) = q.shape[-2:], v.shape[-2:]
        return (dtype in _DTYPES and k.dtype is dtype and v.dtype is dtype and device.type == "cuda"
                and k.device == device and v.device == device and g.device == device and beta.device == device
                and g.dtype is torch.float32 and beta.dtype is torch.float32 and k.shape == q.shape
                and v.shape[:-2] == lead and g.shape == v.shape[:-1] and beta.shape == g.shape
                and 0 < hk <= hv and hv % hk == 0 and 0 < kd <= _native.MAX_KEY_DIM and vd > 0
                and (q.stride(-1) == 1 or kd == 1) and (k.stride(-1) == 1 or kd == 1) and (v.stride(-1) == 1 or vd == 1)
                and (starts is None or (starts.dtype in _MASKS and starts.device == device and starts.shape == lead)))
    except (AttributeError, TypeError, ValueError, IndexError):
        return False


def _check_rule(q, k, v, g, beta, starts, lead: tuple[str, ...]) -> None:
    n = len(lead)
    if _fine_rule(q, k, v, g, beta, starts) and q.dim() == n + 2:
        return
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
    raise RuntimeError("q, k, v, g, beta and starts do not go together")


def _check_state(name: str, state, q, v) -> None:
    want = (q.size(0), v.size(-2), q.size(-1), v.size(-1))
    if (isinstance(state, torch.Tensor) and state.dtype is torch.float32 and state.device == q.device
            and state.shape == want and state.is_contiguous()):
        return
    _check_tensor(name, state, (torch.float32,), 4, q.device)
    _check(tuple(state.shape) == want, f"{name} must be [Envs, ValueHeads, KeyDim, ValueDim] = {list(want)}")
    raise RuntimeError(f"{name} must be contiguous")


# Rollouts of so few steps go token by token: a chunk takes as long for one token as for 64, a step
# as long as its state. Four steps and a chunk on the device, us, with the state returned: 1 x 8 heads
# of 128, 8.6 and 14.4; 64 x 4 of 64, float32, 6.8 and 17.3; 1024 x 4 of 64, 38 and 81; 1024 x 4 of 128,
# 157 and 180. Eight: 14.7 and 14.6; 10.6 and 17.6; 53 and 82; 227 and 182: four is safe for states of
# any size, small ones would gain up to eight.
_STEPWISE = 4

_FARTHEST = ((1 << 31) - 1) // _native.CHUNK - (1 << 18)  # bytes between steps that the chunked kernels reach


def _rows_apart(t: torch.Tensor) -> torch.Tensor:
    """``t`` as the chunked kernels read it: steps that do not overlap (an expanded axis) and lie
    within reach; else a copy."""
    if t.size(1) <= 1 or t.size(3) <= t.stride(1) <= _FARTHEST // t.element_size():
        return t
    return t.contiguous()


def _pack_rule(q, k, v, g, beta, starts, scale, initial_state, out, final_state, matrices=None, scratch=None, states=None,
               updates=None) -> bytes:
    envs, steps, key_heads, key_dim = q.shape
    value_heads, value_dim = v.shape[2:]
    return _native.PACK_RULE(
        _DTYPES[q.dtype], key_heads, value_heads, key_dim, value_dim, envs, steps, scale,
        q.data_ptr(), k.data_ptr(), v.data_ptr(), *q.stride()[:3], *k.stride()[:3], *v.stride()[:3],
        g.data_ptr(), beta.data_ptr(), *g.stride(), *beta.stride(),
        *((0, 0, 0) if starts is None else (starts.data_ptr(), *starts.stride())),
        _ptr(initial_state), out.data_ptr(), _ptr(final_state), _ptr(matrices), _ptr(scratch), _ptr(states), _ptr(updates))


def _forward(q, k, v, g, beta, starts, scale, initial_state, return_state, save):
    """(out, final state or None, matrices, states, updates): the last three for a backward pass."""
    envs, steps, heads, dim = v.shape
    device, key_dim, chunks = v.device, q.size(3), -(-steps // _native.CHUNK)
    floats = dict(dtype=torch.float32, device=device)
    out = torch.empty(v.shape, dtype=v.dtype, device=device)
    state = states = updates = scratch = None
    if return_state:
        state = torch.empty((envs, heads, key_dim, dim), **floats)
    matrices = torch.empty((envs * heads, chunks, _native.CHUNK_MATRICES), **floats)
    if save:
        states = torch.empty((envs * heads, max(0, chunks - 1), key_dim, dim), **floats)
        updates = torch.empty((envs * heads, steps, dim), **floats)
    args = (q, k, v, g, beta, starts, scale, initial_state, out, state, matrices)
    rule = _pack_rule(*args, None, states, updates)
    size = _native.check(_native.lib().navi_delta_scratch(rule))
    if size:
        scratch = torch.empty(size // 4, **floats)
        rule = _pack_rule(*args, scratch, states, updates)
    _call(_native.lib().navi_delta_forward, device, rule)
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
        device = q.device
        d_q, d_k, d_v, d_g, d_beta = (torch.empty(t.shape, dtype=t.dtype, device=device) for t in (q, k, v, g, beta))
        d_state = torch.empty_like(initial_state) if initial_state is not None and ctx.needs_input_grad[5] else None
        if v.numel() == 0:
            if d_state is not None:
                d_state = torch.zeros_like(d_state) if grad_state is None else grad_state.clone()
            return d_q, d_k, d_v, d_g, d_beta, d_state, None, None, None
        rule = _pack_rule(q, k, v, g, beta, starts, ctx.scale, initial_state, grad_out, None, matrices, None, states, updates)
        lib = _native.lib()
        size = _native.check(lib.navi_delta_workspace(rule))
        workspace = torch.empty(size // 4, dtype=torch.float32, device=device)
        gradients = _native.PACK_GRADIENTS(
            grad_out.data_ptr(), *grad_out.stride()[:3], _ptr(grad_state), d_q.data_ptr(), d_k.data_ptr(), d_v.data_ptr(),
            d_g.data_ptr(), d_beta.data_ptr(), _ptr(d_state), workspace.data_ptr())
        _call(lib.navi_delta_backward, device, rule, gradients)
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
        _check_state("initial_state", initial_state, q, v)
    _check_tangents(q, k, v, g, beta, initial_state)
    scale = q.size(-1) ** -0.5 if scale is None else float(scale)
    grad = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or g.requires_grad
                                      or beta.requires_grad or (initial_state is not None and initial_state.requires_grad))
    if not grad and q.size(1) <= _STEPWISE:
        out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
        state = None
        if return_state:
            state = torch.empty((v.size(0), v.size(2), q.size(3), v.size(3)), dtype=torch.float32, device=v.device)
        _call(_native.lib().navi_delta_step, q.device,
              _pack_rule(q, k, v, g, beta, starts, scale, initial_state, out, state))
        return (out, state) if return_state else out
    q, k, v = _rows_apart(q), _rows_apart(k), _rows_apart(v)
    if grad:
        return _DeltaRule.apply(q, k, v, g, beta, initial_state, starts, scale, bool(return_state))
    out, state, *_ = _forward(q, k, v, g, beta, starts, scale, initial_state, return_state, False)
    return (out, state) if return_state else out


def gated_delta_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                     state: torch.Tensor, *, scale: float | None = None, starts: torch.Tensor | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """One token of every environment: ``gated_delta_rule`` without the ``Steps`` axis.

    ``state`` (float32, ``[Envs, ValueHeads, KeyDim, ValueDim]``) is updated in place; the
    output goes to ``out`` (like ``v``, contiguous) if given, which shares no memory with the
    inputs but may be ``v`` itself. Autograd is told of both writes: what has saved either raises
    backward. No gradients: this is the form for acting.
    """
    _check_rule(q, k, v, g, beta, starts, ("Envs",))
    _check_state("state", state, q, v)
    device, written = q.device, [state]
    if out is not None:
        written.append(out)
        _check_tensor("out", out, (v.dtype,), 3, device)
        _check(out.shape == v.shape and out.is_contiguous(), "out must be like v, contiguous")
    _check_tangents(q, k, v, g, beta, state, out)
    if torch.is_grad_enabled():
        _check(not (q.requires_grad or k.requires_grad or v.requires_grad or g.requires_grad or beta.requires_grad
                    or state.requires_grad or (out is not None and out.requires_grad)),
               "gated_delta_step has no gradients; use gated_delta_rule, or torch.no_grad()")
    if out is None:
        out = torch.empty(v.shape, dtype=v.dtype, device=device)
    envs, key_heads, key_dim = q.shape
    (q0, q1, _), (k0, k1, _), (v0, v1, _) = q.stride(), k.stride(), v.stride()
    (g0, g1), (b0, b1), at = g.stride(), beta.stride(), state.data_ptr()
    rule = _native.PACK_RULE(
        _DTYPES[q.dtype], key_heads, v.size(1), key_dim, v.size(2), envs, 1,
        key_dim ** -0.5 if scale is None else float(scale), q.data_ptr(), k.data_ptr(), v.data_ptr(),
        q0, 0, q1, k0, 0, k1, v0, 0, v1, g.data_ptr(), beta.data_ptr(), g0, 0, g1, b0, 0, b1,
        *((0, 0, 0) if starts is None else (starts.data_ptr(), starts.stride(0), 0)),
        at, out.data_ptr(), at, 0, 0, 0, 0)
    _call(_native.lib().navi_delta_step, device, rule)
    _written(written)
    return out


# ---- norms of queries and keys, rotation by position ----


_NORMS = {"rms": _native.NORM_RMS, "l2": _native.NORM_L2}


def _pack_norm(q, k, q_weight, k_weight, cos, sin, positions, norm, eps, interleaved, outputs, backward=(0,) * 13) -> bytes:
    envs, steps, query_heads, dim = q.shape
    end, pairs = (0, 0) if cos is None else cos.shape
    return _native.PACK_NORM(
        _DTYPES[q.dtype], _NORMS[norm], query_heads, k.size(2), dim, pairs, interleaved,
        positions is not None and positions.dtype is torch.int64, envs, steps, eps, q.data_ptr(), k.data_ptr(),
        *q.stride()[:3], *k.stride()[:3], _ptr(q_weight), _ptr(k_weight),
        *((0, 0, 0) if positions is None else (positions.data_ptr(), *positions.stride())), _ptr(cos), _ptr(sin), end,
        *outputs, *backward)


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
        device = q.device
        d_q, d_k = (torch.empty(t.shape, dtype=t.dtype, device=device) for t in (q, k))
        d_weights = [torch.empty_like(w) if w is not None and ctx.needs_input_grad[2 + i] else None
                     for i, w in enumerate((q_weight, k_weight))]
        args = (q, k, q_weight, k_weight, cos, sin, positions, *ctx.rest)
        lib, partial = _native.lib(), None
        if any([w is not None for w in d_weights]):
            size = _native.check(lib.navi_qk_norm_workspace(_pack_norm(*args, (0, 0))))
            partial = torch.empty(size // 4, dtype=torch.float32, device=device)
        packed = _pack_norm(*args, (0, 0), (grad_q.data_ptr(), grad_k.data_ptr(), *grad_q.stride()[:3], *grad_k.stride()[:3],
                                            d_q.data_ptr(), d_k.data_ptr(), _ptr(d_weights[0]), _ptr(d_weights[1]),
                                            _ptr(partial)))
        _call(lib.navi_qk_norm_backward, device, packed)
        return d_q, d_k, d_weights[0], d_weights[1], None, None, None, None, None, None


def _norm_forward(q, k, *rest):
    q_out, k_out = torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty(k.shape, dtype=k.dtype, device=k.device)
    _call(_native.lib().navi_qk_norm, q.device, _pack_norm(q, k, *rest, (q_out.data_ptr(), k_out.data_ptr())))
    return q_out, k_out


def _fine_norm(q, k, q_weight, k_weight, cos, sin, positions, norm) -> bool:
    try:
        device, dtype, (envs, steps, _, dim) = q.device, q.dtype, q.shape
        return (dtype in _DTYPES and k.dtype is dtype and device.type == "cuda" and k.device == device and norm in _NORMS
                and k.dim() == 4 and k.shape[:2] == (envs, steps) and k.size(3) == dim and 0 < dim <= _native.MAX_NORM_DIM
                and (q.stride(3) == 1 or dim == 1) and (k.stride(3) == 1 or dim == 1)
                and all(w is None or (w.dtype is torch.float32 and w.device == device and w.shape == (dim,)
                                      and w.is_contiguous()) for w in (q_weight, k_weight))
                and ((cos is None and sin is None and positions is None)
                     or (cos.dtype is torch.float32 and sin.dtype is torch.float32 and cos.device == device
                         and sin.device == device and cos.dim() == 2 and cos.shape == sin.shape and cos.is_contiguous()
                         and sin.is_contiguous() and cos.size(0) > 0 and 0 < 2 * cos.size(1) <= dim
                         and (positions is None or (positions.dtype in (torch.int32, torch.int64)
                                                    and positions.device == device and positions.shape == (envs, steps))))))
    except (AttributeError, TypeError, ValueError, IndexError):
        return False


def _check_norm(q, k, q_weight, k_weight, cos, sin, positions, norm) -> None:
    if _fine_norm(q, k, q_weight, k_weight, cos, sin, positions, norm):
        return
    _check_tensor("q", q, tuple(_DTYPES), 4)
    _check_tensor("k", k, (q.dtype,), 4, q.device)
    _check(q.shape[:2] == k.shape[:2] and q.size(3) == k.size(3), "q and k must be [Envs, Steps, Heads, HeadDim], alike but for Heads")
    _check(0 < q.size(3) <= _native.MAX_NORM_DIM, f"the head dimension must be in [1, {_native.MAX_NORM_DIM}]")
    _check(_dense_last(q) and _dense_last(k), "q and k must be contiguous in their last dimension")
    _check(norm in _NORMS, "norm must be 'rms' or 'l2'")
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
    raise RuntimeError("q, k, the weights, cos, sin and positions do not go together")


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
    ``cos``, ``sin``: float32 ``[Positions, Pairs]`` tables (without gradients) that rotate the first ``2 * Pairs``
    numbers of a row, pair i being (i, i + Pairs), or (2 i, 2 i + 1) with ``interleaved``.
    ``positions``: ``[Envs, Steps]`` int32 or int64 rows of the tables (a token's step by
    default); one outside the tables gives NaN in the numbers that it would rotate.
    """
    _check_norm(q, k, q_weight, k_weight, cos, sin, positions, norm)
    _check_tangents(q, k, q_weight, k_weight, cos, sin)
    eps = float(eps)
    _check(math.isfinite(eps) and eps >= 0.0, "eps must be finite and not negative")
    args = (q, k, q_weight, k_weight, cos, sin, positions, norm, eps, bool(interleaved))
    if cos is not None and torch.is_grad_enabled():
        _check(not (cos.requires_grad or sin.requires_grad), "cos and sin have no gradients; detach them")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or (q_weight is not None and q_weight.requires_grad)
                                    or (k_weight is not None and k_weight.requires_grad)):
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
    an optimizer's flat buffer, for one). Tensors that are written share no memory with others (a
    parameter that is used twice is named once). A norm that is not finite spoils the gradients as
    the formula says: NaN gives NaN, infinity gives 0 (NaN where the gradient is infinite).
    """
    max_norm, eps = float(max_norm), float(eps)
    _check(max_norm >= 0.0 and eps >= 0.0, "max_norm and eps must not be negative")
    grads = list(grads)
    to = grads if out is None else list(out)
    _check(len(to) == len(grads), "out must be as long as grads")
    if any([x is None for x in grads]):
        to = [y for x, y in zip(grads, to) if x is not None]
        grads = [x for x in grads if x is not None]
    _check(len(grads) > 0, "grads must hold at least one tensor")
    if not _fine_grads(grads, to):
        _check_grads(grads, to)
    _check_tangents(*grads, *to)
    n, device = len(grads), grads[0].device
    norm = torch.empty((), dtype=torch.float32, device=device)
    partial = torch.empty(_native.NORM_PARTIALS, dtype=torch.float32, device=device)
    at = struct.pack(f"{n}P", *[x.data_ptr() for x in grads])
    _call(_native.lib().navi_clip_grad_norm, device,
          n, at, at if to is grads else struct.pack(f"{n}P", *[y.data_ptr() for y in to]),
          struct.pack(f"{n}q", *[x.numel() for x in grads]), struct.pack(f"{n}i", *[_DTYPES[x.dtype] for x in grads]),
          max_norm, eps, norm.data_ptr(), partial.data_ptr())
    _written(to)
    return norm


def _fine_grads(grads: list, to: list) -> bool:
    """Whether all are contiguous and alike: what nearly every call brings."""
    try:
        device = grads[0].get_device()
        return (device >= 0 and all([x.is_contiguous() and x.get_device() == device and x.dtype in _DTYPES for x in grads])
                and (to is grads or all([y.is_contiguous() and y.get_device() == device and y.dtype is x.dtype
                                         and y.shape == x.shape for x, y in zip(grads, to)])))
    except (AttributeError, TypeError, RuntimeError):
        return False


def _check_grads(grads: list, to: list) -> None:
    for x, y in zip(grads, to):
        _check(isinstance(x, torch.Tensor) and x.is_cuda and x.layout == torch.strided, "grads must be dense CUDA tensors")
        _check(x.dtype in _DTYPES, "grads must be float32, bfloat16 or float16")
        _check(x.device == grads[0].device, "grads must be on one device")
        _check(x.is_contiguous() or torch.ops.aten.is_non_overlapping_and_dense(x), "grads must fill their memory without gaps")
        if y is not x:
            _check(isinstance(y, torch.Tensor) and y.dtype == x.dtype and y.shape == x.shape and y.device == x.device
                   and (y.is_contiguous() if x.is_contiguous() else y.stride() == x.stride()),
                   "out must be like grads in shapes, types, strides and device")

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
* ``selective_scan`` / ``selective_scan_step``: a memory of one ``StateDim x HeadDim`` matrix per head
  that forgets at a rate that each token chooses, ``S <- exp(beta a) S + beta b x^T``, ``y = S^T c + d x``
  with ``beta = softplus(dt + dt_bias)``; ``causal_conv`` / ``causal_conv_step``: the short convolution
  over the last frames that stands before it. Each with gradients over rollouts and for one frame.
* ``block_norm``: what stands between two blocks of a residual stream, the norm after the one, its gate
  and scale, the sum, and the norm before the next, in one pass.
* ``orthogonalize``: the updates of weight matrices made nearly orthogonal by Newton-Schulz products.

The kernels run on PyTorch's current stream, never wait for the device and keep nothing of a
call; queries, keys and values (``x``, ``b`` and ``c``) may be views of one projection (any strides
but the last axis's). Misuse raises ``RuntimeError``, forward-mode derivatives do too; there is no CPU fallback.
"""

from __future__ import annotations

import math
import struct
from typing import Iterable

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _policy_native as _native

__all__ = ["gated_delta_rule", "gated_delta_step", "qk_norm", "clip_grad_norm", "causal_conv", "causal_conv_step",
           "selective_scan", "selective_scan_step", "block_norm", "orthogonalize"]

_DTYPES = {torch.float32: _native.F32, torch.bfloat16: _native.BF16, torch.float16: _native.F16}
_MASKS = (torch.bool, torch.uint8)
_MOST = torch.finfo(torch.float32).max

# Arguments are looked over twice: `_fine` in one expression on every call (a call of one frame
# is bound by the host), and by name, for the message, where that found something. Where a call of
# one frame or of a few rows takes the device less time than its arguments take Python, the
# extension `_native.calls` makes it whole, if it is in order (and a frame's asks for no gradients); a
# call that it leaves (None) goes the way below. Allocation, launch and gradients of a block's operators
# are its work too.


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


def _check_plain(*tensors) -> None:
    """Memory holds what a tensor shows (that of a lazily negated view holds its negative)."""
    _check(not any([t is not None and t.is_neg() for t in tensors]), "lazily negated views are not taken: resolve_neg() them")


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


# ---- a selective state space scan ----


def _fine_vectors(device, *wanted) -> bool:
    """Whether each (vector or None, length) is a dense float32 vector of the device."""
    for t, n in wanted:
        if t is not None and not (t.dtype is torch.float32 and t.device == device and t.shape == (n,) and t.is_contiguous()):
            return False
    return True


def _check_vector(name: str, t, length: int, what: str, device) -> None:
    if t is None:
        return
    _check_tensor(name, t, (torch.float32,), 1, device)
    _check(t.size(0) == length and t.is_contiguous(), f"{name} must be [{what}], contiguous")


def _fine_scan(x, dt, a, b, c, d, dt_bias, starts) -> bool:
    """Whether the inputs are in order ([Envs, Steps, ...] and [Envs, ...] alike)."""
    try:
        lead, device, dtype = x.shape[:-2], x.device, x.dtype
        (heads, head_dim), (groups, state_dim) = x.shape[-2:], b.shape[-2:]
        return (dtype in _DTYPES and b.dtype is dtype and c.dtype is dtype and device.type == "cuda" and b.device == device
                and c.device == device and dt.device == device and dt.dtype is torch.float32 and dt.shape == x.shape[:-1]
                and b.shape[:-2] == lead and c.shape == b.shape and 0 < groups <= heads <= _native.MAX_HEADS and heads % groups == 0
                and 0 < head_dim <= _native.MAX_STATE_DIM and 0 < state_dim <= _native.MAX_STATE_DIM
                and (x.stride(-1) == 1 or head_dim == 1) and (b.stride(-1) == 1 or state_dim == 1)
                and (c.stride(-1) == 1 or state_dim == 1) and a is not None
                and _fine_vectors(device, (a, heads), (d, heads), (dt_bias, heads))
                and (starts is None or (starts.dtype in _MASKS and starts.device == device and starts.shape == lead)))
    except (AttributeError, TypeError, ValueError, IndexError):
        return False


def _check_scan(x, dt, a, b, c, d, dt_bias, starts, lead: tuple[str, ...]) -> None:
    n = len(lead)
    if _fine_scan(x, dt, a, b, c, d, dt_bias, starts) and x.dim() == n + 2:
        return
    shape = ", ".join(lead)
    _check(isinstance(x, torch.Tensor) and x.is_cuda, "x must be a CUDA tensor")
    _check_tensor("x", x, tuple(_DTYPES), n + 2)
    for name, t in (("b", b), ("c", c)):
        _check_like("x", name, t, (x.dtype,), n + 2, x.device)
    _check_like("x", "dt", dt, (torch.float32,), n + 1, x.device)
    for name, t in (("x", x), ("b", b), ("c", c)):
        _check(_dense_last(t), f"{name} must be contiguous in its last dimension")
    _check(b.shape == c.shape and b.shape[:n] == x.shape[:n], f"b and c must both be [{shape}, Groups, StateDim]")
    heads, groups = x.size(n), b.size(n)
    _check(heads > 0 and groups > 0 and heads % groups == 0, "the heads must be a multiple of the groups")
    _check(heads <= _native.MAX_HEADS, f"the heads must be at most {_native.MAX_HEADS}")
    _check(0 < x.size(-1) <= _native.MAX_STATE_DIM and 0 < b.size(-1) <= _native.MAX_STATE_DIM,
           f"the head and state dimensions must be in [1, {_native.MAX_STATE_DIM}]")
    _check(dt.shape == x.shape[:-1], f"dt must be [{shape}, Heads]")
    _check(isinstance(a, torch.Tensor), "a must be a CUDA tensor")
    for name, t in (("a", a), ("d", d), ("dt_bias", dt_bias)):
        _check_vector(name, t, heads, "Heads", x.device)
    if starts is not None:
        _check_like("x", "starts", starts, _MASKS, n, x.device)
        _check(starts.shape == x.shape[:n], f"starts must be [{shape}]")
    raise RuntimeError("x, dt, a, b, c, d, dt_bias and starts do not go together")


def _check_like(of: str, name: str, t, dtypes, dims: int, device) -> None:
    _check(isinstance(t, torch.Tensor) and t.is_cuda, f"{name} must be a CUDA tensor")
    _check(t.device == device, f"{name} must be on the same device as {of} ({device})")
    _check_tensor(name, t, dtypes, dims)


def _check_scan_state(name: str, state, x, b) -> None:
    want = (x.size(0), x.size(-2), b.size(-1), x.size(-1))
    if (isinstance(state, torch.Tensor) and state.dtype is torch.float32 and state.device == x.device
            and state.shape == want and state.is_contiguous()):
        return
    _check_like("x", name, state, (torch.float32,), 4, x.device)
    _check(tuple(state.shape) == want, f"{name} must be [Envs, Heads, StateDim, HeadDim] = {list(want)}")
    raise RuntimeError(f"{name} must be contiguous")


def selective_scan(x: torch.Tensor, dt: torch.Tensor, a: torch.Tensor, b: torch.Tensor, c: torch.Tensor, *,
                   d: torch.Tensor | None = None, dt_bias: torch.Tensor | None = None, starts: torch.Tensor | None = None,
                   initial_state: torch.Tensor | None = None, return_state: bool = False):
    """A selective state space scan over whole rollouts, differentiable in everything but ``starts``.

    Per head, with ``beta = softplus(dt + dt_bias)`` and a state ``S`` of ``StateDim x HeadDim``
    numbers: ``S <- exp(beta a) S + beta b x^T``, ``y = S^T c + d x``.
    ``x``: ``[Envs, Steps, Heads, HeadDim]`` in float32, bfloat16 or float16, ``b``, ``c``:
    ``[Envs, Steps, Groups, StateDim]`` of the same type, with ``Heads`` a multiple of ``Groups``
    (head h reads group ``h // (Heads // Groups)``) and at most 16384; both dimensions up to 128. ``dt``:
    ``[Envs, Steps, Heads]`` float32; ``a`` (rates, at most 0), ``d`` and ``dt_bias`` (zeros by
    default): ``[Heads]`` float32. ``starts``: ``[Envs, Steps]`` bool or uint8, tokens that begin an
    episode: the state before one is forgotten (at the first step, whatever it holds).
    ``initial_state``: ``[Envs, Heads, StateDim, HeadDim]`` float32, zeros by default.

    Returns ``y`` like ``x``, with ``return_state`` also the state after the last token.
    Arithmetic is of float32's precision for every type, rounded once at the end. A NaN or
    infinity in the inputs may reach every token of its chunk of 64 tokens and what follows
    them, beyond the start of an episode too.
    """
    return_state = bool(return_state)
    if forward_ad._current_level < 0:
        done = _native.calls.selective_scan(x, dt, a, b, c, d, dt_bias, initial_state, starts, return_state, _STEPWISE)
        if done is not None:
            return done
    _check_scan(x, dt, a, b, c, d, dt_bias, starts, ("Envs", "Steps"))
    if initial_state is not None:
        _check_scan_state("initial_state", initial_state, x, b)
    _check_tangents(x, dt, a, b, c, d, dt_bias, initial_state)
    # (rollouts of few steps without gradients go token by token, as for the gated delta rule)
    return _native.calls.scan(x, dt, a, b, c, d, dt_bias, initial_state, starts, return_state, _STEPWISE)


def selective_scan_step(x: torch.Tensor, dt: torch.Tensor, a: torch.Tensor, b: torch.Tensor, c: torch.Tensor,
                        state: torch.Tensor, *, d: torch.Tensor | None = None, dt_bias: torch.Tensor | None = None,
                        starts: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """One token of every environment: ``selective_scan`` without the ``Steps`` axis.

    ``state`` (float32, ``[Envs, Heads, StateDim, HeadDim]``) is updated in place; the output
    goes to ``out`` (like ``x``, contiguous) if given, which shares no memory with the inputs but
    may be ``x`` itself. Autograd is told of both writes: what has saved either raises backward.
    No gradients: this is the form for acting.
    """
    if forward_ad._current_level < 0:
        done = _native.calls.selective_step(x, dt, a, b, c, state, d, dt_bias, starts, out)
        if done is not None:
            return done
    _check_scan(x, dt, a, b, c, d, dt_bias, starts, ("Envs",))
    _check_scan_state("state", state, x, b)
    written = [state]
    if out is not None:
        written.append(out)
        _check_like("x", "out", out, (x.dtype,), 3, x.device)
        _check(out.shape == x.shape and out.is_contiguous(), "out must be like x, contiguous")
    inputs = (x, dt, a, b, c, d, dt_bias, state, out)
    _check_tangents(*inputs)
    if torch.is_grad_enabled():
        _check(not any([t is not None and t.requires_grad for t in inputs]),
               "selective_scan_step has no gradients; use selective_scan, or torch.no_grad()")
    _check_plain(*inputs)
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    envs, heads, head_dim = x.shape
    (x0, x1, _), (b0, b1, _), (c0, c1, _), at = x.stride(), b.stride(), c.stride(), state.data_ptr()
    packed = _native.PACK_SCAN(
        _DTYPES[x.dtype], heads, b.size(1), b.size(2), head_dim, envs, 1, x.data_ptr(), b.data_ptr(), c.data_ptr(),
        x0, 0, x1, b0, 0, b1, c0, 0, c1, dt.data_ptr(), dt.stride(0), 0, dt.stride(1), a.data_ptr(), _ptr(d), _ptr(dt_bias),
        *((0, 0, 0) if starts is None else (starts.data_ptr(), starts.stride(0), 0)), at, out.data_ptr(), at, 0,
        0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
    _call(_native.lib().navi_selective_step, x.device, packed)
    _written(written)
    return out


# ---- a short convolution over the last frames ----


_ACTIVATIONS = {"silu": _native.ACT_SILU, None: _native.ACT_NONE}


def _number_of(activation) -> int | None:
    return _ACTIVATIONS.get(activation) if activation is None or isinstance(activation, str) else None


def _fine_conv(x, weight, bias, starts, activation) -> bool:
    try:
        channels, device = x.size(-1), x.device
        return (x.dtype in _DTYPES and device.type == "cuda" and (x.stride(-1) == 1 or channels == 1) and 0 < channels <= 65536
                and weight.dtype is torch.float32 and weight.device == device and weight.dim() == 2
                and weight.size(0) == channels and 2 <= weight.size(1) <= _native.MAX_TAPS and weight.is_contiguous()
                and _fine_vectors(device, (bias, channels)) and _number_of(activation) is not None
                and (starts is None or (starts.dtype in _MASKS and starts.device == device and starts.shape == x.shape[:-1])))
    except (AttributeError, TypeError, ValueError, IndexError, RuntimeError):
        return False


def _check_conv(x, weight, bias, starts, activation, lead: tuple[str, ...]) -> None:
    n = len(lead)
    if _fine_conv(x, weight, bias, starts, activation) and x.dim() == n + 1:
        return
    shape = ", ".join(lead)
    _check(isinstance(x, torch.Tensor) and x.is_cuda, "x must be a CUDA tensor")
    _check_tensor("x", x, tuple(_DTYPES), n + 1)
    _check(_dense_last(x), "x must be contiguous in its last dimension")
    _check(0 < x.size(-1) <= 65536, "the channels must be in [1, 65536]")
    _check_like("x", "weight", weight, (torch.float32,), 2, x.device)
    _check(weight.size(0) == x.size(-1) and 2 <= weight.size(1) <= _native.MAX_TAPS and weight.is_contiguous(),
           f"weight must be [Channels, Taps], contiguous, with 2 to {_native.MAX_TAPS} taps")
    _check_vector("bias", bias, x.size(-1), "Channels", x.device)
    if starts is not None:
        _check_like("x", "starts", starts, _MASKS, n, x.device)
        _check(starts.shape == x.shape[:-1], f"starts must be [{shape}]")
    _check(_number_of(activation) is not None, "activation must be 'silu' or None")
    raise RuntimeError("x, weight, bias and starts do not go together")


def _check_window(name: str, window, x, weight) -> None:
    want = (x.size(0), weight.size(1) - 1, x.size(-1))
    if (isinstance(window, torch.Tensor) and window.dtype is x.dtype and window.device == x.device
            and window.shape == want and window.is_contiguous()):
        return
    _check_like("x", name, window, (x.dtype,), 3, x.device)
    _check(tuple(window.shape) == want, f"{name} must be [Envs, Taps - 1, Channels] = {list(want)}")
    raise RuntimeError(f"{name} must be contiguous")


def causal_conv(x: torch.Tensor, weight: torch.Tensor, *, bias: torch.Tensor | None = None,
                starts: torch.Tensor | None = None, initial_window: torch.Tensor | None = None,
                return_window: bool = False, activation: str | None = "silu"):
    """A short convolution over the last frames of a rollout, channel by channel; differentiable in
    x, weight, bias and initial_window.

    ``y[t] = act(bias + sum_j weight[:, j] x[t - (Taps - 1) + j])``. ``x``: ``[Envs, Steps, Channels]``
    in float32, bfloat16 or float16; ``weight``: ``[Channels, Taps]`` float32 with 2 to 4 taps;
    ``bias``: ``[Channels]`` float32. ``activation``: ``"silu"`` or None. ``starts``: ``[Envs, Steps]``
    bool or uint8, tokens that begin an episode: inputs before one count as zeros for it and what
    follows, whatever they hold. ``initial_window``: ``[Envs, Taps - 1, Channels]`` like ``x``, the
    inputs before the first step (zeros by default).

    Returns ``y`` like ``x``, with ``return_window`` also the window after the last step: its last
    ``Taps - 1`` inputs, zeros in place of those of an earlier episode. Sums are float32's, rounded
    once at the end.
    """
    return_window, number = bool(return_window), _number_of(activation)
    if forward_ad._current_level < 0:
        done = _native.calls.causal_conv(x, weight, bias, initial_window, starts, number, return_window)
        if done is not None:
            return done
    _check_conv(x, weight, bias, starts, activation, ("Envs", "Steps"))
    if initial_window is not None:
        _check_window("initial_window", initial_window, x, weight)
    inputs = (x, weight, bias, initial_window)
    _check_tangents(*inputs)
    return _native.calls.conv(*inputs, starts, number, return_window)


def causal_conv_step(x: torch.Tensor, weight: torch.Tensor, window: torch.Tensor, *, bias: torch.Tensor | None = None,
                     starts: torch.Tensor | None = None, activation: str | None = "silu",
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """One frame of every environment: ``causal_conv`` without the ``Steps`` axis.

    ``window`` (``[Envs, Taps - 1, Channels]`` like ``x``) is updated in place; the output goes to
    ``out`` (like ``x``, contiguous) if given, which shares no memory with the inputs but may be
    ``x`` itself. Autograd is told of both writes. No gradients: this is the form for acting.
    """
    if forward_ad._current_level < 0:
        done = _native.calls.conv_step(x, weight, window, bias, starts, _number_of(activation), out)
        if done is not None:
            return done
    _check_conv(x, weight, bias, starts, activation, ("Envs",))
    _check_window("window", window, x, weight)
    written = [window]
    if out is not None:
        written.append(out)
        _check_like("x", "out", out, (x.dtype,), 2, x.device)
        _check(out.shape == x.shape and out.is_contiguous(), "out must be like x, contiguous")
    inputs = (x, weight, bias, window, out)
    _check_tangents(*inputs)
    if torch.is_grad_enabled():
        _check(not any([t is not None and t.requires_grad for t in inputs]),
               "causal_conv_step has no gradients; use causal_conv, or torch.no_grad()")
    _check_plain(*inputs)
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    at = window.data_ptr()
    packed = _native.PACK_CONV(
        _DTYPES[x.dtype], x.size(1), weight.size(1), _ACTIVATIONS[activation], x.size(0), 1, x.data_ptr(), x.stride(0), 0,
        weight.data_ptr(), _ptr(bias), *((0, 0, 0) if starts is None else (starts.data_ptr(), starts.stride(0), 0)),
        at, out.data_ptr(), at, 0, 0, 0, 0, 0, 0, 0, 0, 0)
    _call(_native.lib().navi_causal_conv, x.device, packed)
    _written(written)
    return out


# ---- between two blocks of a residual stream ----


def _fine_block(y, residual, gate, scale, post_weight, pre_weight) -> bool:
    try:
        device, dtype, width = y.device, y.dtype, y.size(-1)
        return (dtype in _DTYPES and device.type == "cuda" and y.dim() == 3 and residual.device == device
                and (residual.dtype is dtype or residual.dtype is torch.float32) and residual.shape == y.shape
                and 0 < width <= _native.MAX_BLOCK_WIDTH and (width == 1 or (y.stride(2) == 1 and residual.stride(2) == 1))
                and (gate is None or (gate.dtype is dtype and gate.device == device and gate.shape == y.shape
                                      and (gate.stride(2) == 1 or width == 1)))
                and _fine_vectors(device, (scale, width), (post_weight, width), (pre_weight, width)))
    except (AttributeError, TypeError, ValueError, IndexError, RuntimeError):
        return False


def _check_block(y, residual, gate, scale, post_weight, pre_weight) -> None:
    if _fine_block(y, residual, gate, scale, post_weight, pre_weight):
        return
    _check(isinstance(y, torch.Tensor) and y.is_cuda, "y must be a CUDA tensor")
    _check_tensor("y", y, tuple(_DTYPES), 3)
    _check_like("y", "residual", residual, tuple({y.dtype, torch.float32}), 3, y.device)
    _check(residual.shape == y.shape, "residual must be [Envs, Steps, Width] like y")
    if gate is not None:
        _check_like("y", "gate", gate, (y.dtype,), 3, y.device)
        _check(gate.shape == y.shape, "gate must be [Envs, Steps, Width] like y")
    for name, t in (("y", y), ("residual", residual), ("gate", gate)):
        _check(t is None or _dense_last(t), f"{name} must be contiguous in its last dimension")
    _check(0 < y.size(2) <= _native.MAX_BLOCK_WIDTH, f"the width must be in [1, {_native.MAX_BLOCK_WIDTH}]")
    for name, t in (("scale", scale), ("post_weight", post_weight), ("pre_weight", pre_weight)):
        _check_vector(name, t, y.size(2), "Width", y.device)
    raise RuntimeError("y, residual, gate, scale and the weights do not go together")


def block_norm(y: torch.Tensor, residual: torch.Tensor, *, gate: torch.Tensor | None = None,
               scale: torch.Tensor | None = None, post_weight: torch.Tensor | None = None,
               pre_weight: torch.Tensor | None = None, eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """What stands between two blocks of a residual stream, in one pass: the norm after a block, its
    gate and scale, the sum with the stream, and the norm before the next block; differentiable in
    everything.

    ``stream = residual + scale * norm(y) * post_weight * silu(gate)`` and ``normed = norm(stream) *
    pre_weight``, with ``norm(x) = x / sqrt(mean(x^2) + eps)`` over the last axis; what is not given
    is left out. ``y`` (the block's output) and ``gate``: ``[Envs, Steps, Width]`` in float32, bfloat16 or
    float16, width up to 8192; ``residual``: the stream before, of the same type or float32;
    ``scale``, ``post_weight``, ``pre_weight``: ``[Width]`` float32. Returns ``stream`` like
    ``residual`` and ``normed`` like ``y``; ``normed`` is that of the sum before it is rounded.
    """
    eps = float(eps)
    if 0.0 <= eps <= _MOST and forward_ad._current_level < 0:
        done = _native.calls.block_norm(y, residual, gate, scale, post_weight, pre_weight, eps)
        if done is not None:
            return done
    _check_block(y, residual, gate, scale, post_weight, pre_weight)
    _check(0.0 <= eps <= _MOST, "eps must be finite (in float32) and not negative")
    inputs = (y, residual, gate, scale, post_weight, pre_weight)
    _check_tangents(*inputs)
    return _native.calls.block(*inputs, eps)


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


# ---- orthogonal updates ----


_NEWTON = (3.4445, -4.775, 2.0315)


def orthogonalize(updates: Iterable[torch.Tensor | None], *, steps: int = 5,
                  factors: tuple[float, float, float] = _NEWTON, eps: float = 1e-6,
                  out: Iterable[torch.Tensor | None] | None = None) -> None:
    """Makes matrices nearly orthogonal by Newton-Schulz products, as an optimizer's update of weight
    matrices: ``X = G / (|G| + eps)`` (``|G|`` the root of the sum of squares), then ``steps``
    times ``X <- a X + (b A + c A A) X`` with ``A = X X^T`` and ``(a, b, c) = factors``, where ``X`` is
    ``G`` or its transpose, the one with no more rows than columns. With the default factors the
    singular values come out between 0.7 and 1.2.

    ``updates``: float32, bfloat16 and float16 matrices of one device in any mix of sizes and types
    (None is skipped), each contiguous along its rows or its columns; they are replaced, or the
    results go to ``out``, tensors of the same shapes (of any of these types and any strides that do
    not overlap). Tensors that are written share no memory with others. Products are of two float16
    each, of float32's precision, but for bfloat16 results of matrices with more than 256 rows and columns: those
    take products of one float16 (3 to 7 parts in 10^4 of the result before its rounding, which leaves 16; who
    wants less gives a float32 ``out``). Factors that can take singular values ``s`` past 7.9 before the last step, or
    ``b s^2 + c s^4`` past 62 in one, are refused (from ``s = 1`` on; the products' operands hold no more). A
    matrix that holds an infinity or NaN comes out without meaning.
    """
    steps, eps = int(steps), float(eps)
    a, b, c = (float(x) for x in factors)
    _check(1 <= steps <= 100, "steps must be in [1, 100]")
    _check(0.0 <= eps <= _MOST, "eps must be finite (in float32) and not negative")
    _check(max(abs(a), abs(b), abs(c)) <= _MOST, "factors must be finite (in float32)")
    updates = list(updates)
    to = updates if out is None else list(out)
    _check(len(to) == len(updates), "out must be as long as updates")
    if any([x is None for x in updates]):
        to = [y for x, y in zip(updates, to) if x is not None]
        updates = [x for x in updates if x is not None]
    _check(len(updates) > 0, "updates must hold at least one matrix")
    _check_matrices(updates, to)
    _check_tangents(*updates, *to)
    if torch.is_grad_enabled():
        _check(not any([x.requires_grad for x in updates]) and (to is updates or not any([y.requires_grad for y in to])),
               "orthogonalize has no gradients; use torch.no_grad()")
    _check_plain(*updates, *(() if to is updates else to))
    n, device = len(updates), updates[0].device
    packed = b"".join([_native.PACK_MATRIX(x.data_ptr(), y.data_ptr(), *x.shape, *_strides_of(x), *_strides_of(y),
                                           _DTYPES[x.dtype], _DTYPES[y.dtype]) for x, y in zip(updates, to)])
    lib = _native.lib()
    size = _native.check(lib.navi_orthogonalize_workspace(n, packed))
    workspace = torch.empty(size, dtype=torch.uint8, device=device)
    _call(lib.navi_orthogonalize, device, n, packed, steps, a, b, c, eps, workspace.data_ptr())
    _written(to)


def _strides_of(x: torch.Tensor) -> tuple[int, int]:
    """A matrix's strides, those of axes of one as in a contiguous one."""
    r, c = x.stride()
    return (r if x.size(0) > 1 else (x.size(1) if c == 1 else 1), c if x.size(1) > 1 else (1 if r != 1 or x.size(0) <= 1 else x.size(0)))


def _check_matrices(updates: list, to: list) -> None:
    try:
        device = updates[0].get_device()
        if device >= 0 and all([x.dim() == 2 and x.get_device() == device and x.dtype in _DTYPES and x.is_contiguous() for x in updates]) and (
                to is updates or all([y.get_device() == device and y.dtype in _DTYPES and y.shape == x.shape and y.is_contiguous()
                                      for x, y in zip(updates, to)])):
            return
    except (AttributeError, TypeError, RuntimeError):
        pass
    for x, y in zip(updates, to):
        _check(isinstance(x, torch.Tensor) and x.is_cuda and x.layout == torch.strided, "updates must be dense CUDA tensors")
        _check(x.dim() == 2, "updates must be matrices")
        _check(x.dtype in _DTYPES, "updates must be float32, bfloat16 or float16")
        _check(x.device == updates[0].device, "updates must be on one device")
        _check(1 in _strides_of(x) or x.numel() == 0, "updates must be contiguous along their rows or columns")
        if y is not x:
            _check(isinstance(y, torch.Tensor) and y.is_cuda and y.layout == torch.strided and y.dtype in _DTYPES
                   and y.shape == x.shape and y.device == x.device,
                   "out must be like updates in shapes and device, float32, bfloat16 or float16")
        _check(y.numel() == 0 or _apart_elements(y), "what is written must not overlap itself")


def _apart_elements(x: torch.Tensor) -> bool:
    (m, n), (r, c) = x.shape, _strides_of(x)
    return (c >= 1 and r >= (n - 1) * c + 1) or (r >= 1 and c >= (m - 1) * r + 1)

"""The policy operators' C entry points refuse arrays that are not aligned to their elements
(addresses that are never read, no GPU)."""

from __future__ import annotations

import ctypes

import pytest

native = pytest.importorskip("navi_amd._policy_native")

TYPED = ("q", "k", "v", "out")
FLOATS = ("g", "beta", "initial_state", "final_state", "states", "updates")


def rule(dtype):
    a = native.DeltaRule(dtype=dtype, key_heads=1, value_heads=1, key_dim=16, value_dim=16, envs=1, steps=100, scale=1.0)
    for name in TYPED + FLOATS + ("matrices",):
        setattr(a, name, 4096)  # never read: every call here is refused before a launch
    for name in ("q", "k", "v"):
        setattr(a, name + "_stride", (ctypes.c_int64 * 3)(1600, 16, 16))
    return a


def refused(code):
    return code == native.NAVI_POLICY_E_ARG and "aligned to their elements" in native.last_error()


@pytest.mark.parametrize("dtype, bytes_each", [(native.F32, 4), (native.BF16, 2), (native.F16, 2)])
def test_rule(dtype, bytes_each):
    lib = native.lib()
    for name in TYPED + FLOATS:
        a = rule(dtype)
        setattr(a, name, 4096 + (bytes_each // 2 if name in TYPED else 2))
        assert refused(lib.navi_delta_forward(ctypes.byref(a), None)), name
        assert refused(lib.navi_delta_step(ctypes.byref(a), None)), name
    for name in ("grad_out", "d_q", "d_k", "d_v", "grad_final_state", "d_g", "d_beta", "d_initial_state"):
        d = native.DeltaGradients(grad_out_stride=(ctypes.c_int64 * 3)(1600, 16, 16))
        for each, _ in d._fields_:
            if each != "grad_out_stride":
                setattr(d, each, 4096)
        setattr(d, name, 4096 + (bytes_each // 2 if name in ("grad_out", "d_q", "d_k", "d_v") else 2))
        assert refused(lib.navi_delta_backward(ctypes.byref(rule(dtype)), ctypes.byref(d), None)), name


@pytest.mark.parametrize("dtype, bytes_each", [(native.F32, 4), (native.BF16, 2), (native.F16, 2)])
def test_norm(dtype, bytes_each):
    lib = native.lib()
    for name in ("q", "k", "q_out", "k_out", "grad_q", "grad_k", "d_q", "d_k", "q_weight", "k_weight", "d_q_weight",
                 "d_k_weight", "partial", "cos", "sin", "positions"):
        a = native.QkNorm(dtype=dtype, query_heads=1, key_heads=1, head_dim=64, pairs=8, positions_wide=1, envs=1, steps=1,
                          positions_end=1)
        for each, kind in a._fields_:
            if kind is ctypes.c_void_p:
                setattr(a, each, 4096)
        typed = name in ("q", "k", "q_out", "k_out", "grad_q", "grad_k", "d_q", "d_k")
        setattr(a, name, 4096 + (bytes_each // 2 if typed else 4 if name == "positions" else 2))
        call = lib.navi_qk_norm if name in ("q_out", "k_out") else lib.navi_qk_norm_backward
        assert refused(call(ctypes.byref(a), None)), name


def test_clip():
    one = lambda kind, x: (kind * 1)(x)  # noqa: E731
    for dtype, odd in ((native.F32, 2), (native.BF16, 1), (native.F16, 1)):
        for at in ((4096 + odd, 8192), (4096, 8192 + odd)):
            code = native.lib().navi_clip_grad_norm(1, *(one(ctypes.c_void_p, p) for p in at), one(ctypes.c_int64, 4),
                                                    one(ctypes.c_int32, dtype), 1.0, 1e-6, 4096, 4096, None)
            assert code == native.NAVI_POLICY_E_ARG and "aligned to its elements" in native.last_error()

"""The gated delta rule's C entry points refuse outputs that share memory with what other workgroups
read, before any launch (addresses that are never read, no GPU)."""

from __future__ import annotations

import ctypes

import pytest

native = pytest.importorskip("navi_amd._policy_native")

ENVS, HEADS, DIM = 3, 2, 16
ROW = HEADS * DIM  # numbers of an environment's frame
STATE = HEADS * DIM * DIM * 4  # bytes of an environment's state
NAMES = ("q", "k", "v", "g", "beta", "starts", "initial_state", "out", "final_state")
AT = {n: (1 + i) << 20 for i, n in enumerate(NAMES)}


def rule(steps, **over):
    a = native.DeltaRule(dtype=native.BF16, key_heads=HEADS, value_heads=HEADS, key_dim=DIM, value_dim=DIM, envs=ENVS,
                         steps=steps, scale=1.0, matrices=64 << 20)
    for name in ("q", "k", "v"):
        setattr(a, name + "_stride", (ctypes.c_int64 * 3)(steps * ROW, ROW, DIM))
    for name in ("g", "beta"):
        setattr(a, name + "_stride", (ctypes.c_int64 * 3)(steps * HEADS, HEADS, 1))
    a.starts_stride = (ctypes.c_int64 * 2)(steps, 1)
    for name, value in {**AT, **over}.items():
        setattr(a, name, value)
    return a


def bytes_of(name, steps):
    if name.endswith("state"):
        return ENVS * STATE
    return ENVS * steps * {"g": 4 * HEADS, "beta": 4 * HEADS, "starts": 1}.get(name, 2 * ROW)


@pytest.mark.parametrize("entry, steps", [("navi_delta_step", 1), ("navi_delta_step", 3), ("navi_delta_forward", 70)])
@pytest.mark.parametrize("written", ["out", "final_state"])
@pytest.mark.parametrize("read", NAMES[:7])
def test_shared_memory_is_refused(entry, steps, written, read):
    ends = bytes_of(read, steps) // 4 * 4 - 4, 4 - bytes_of(written, steps)  # in its last word, in its first
    places = [AT[read] + end for end in ends]
    if (written, read) != ("out", "v"):
        places.append(AT[read])
    if (written, read) == ("final_state", "initial_state") and entry == "navi_delta_step":
        places.remove(AT[read])  # in place
    for place in places:
        code = getattr(native.lib(), entry)(ctypes.byref(rule(steps, **{written: place})), None)
        assert code == native.NAVI_POLICY_E_ARG and "shares memory" in native.last_error(), hex(place)


@pytest.mark.parametrize("entry, steps", [("navi_delta_step", 1), ("navi_delta_forward", 70)])
def test_outputs_that_share_memory_are_refused(entry, steps):
    call = getattr(native.lib(), entry)
    assert call(ctypes.byref(rule(steps, final_state=AT["out"])), None) == native.NAVI_POLICY_E_ARG
    assert "shares memory" in native.last_error()
    # v itself, but not as out lies: heads before environments
    a = rule(steps, out=AT["v"])
    a.v_stride = (ctypes.c_int64 * 3)(steps * DIM, DIM, ENVS * steps * DIM)
    assert call(ctypes.byref(a), None) == native.NAVI_POLICY_E_ARG and "shares memory" in native.last_error()

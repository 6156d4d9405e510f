"""The policy operators' boundary without a GPU: the C ABI's structures and argument checks
(``include/policy/navi_policy.h``) and what the Python layer refuses before any launch."""

from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from . import policy_reference as ref

ROOT = Path(__file__).resolve().parents[1]
native = pytest.importorskip("navi_amd._policy_native")
policy = pytest.importorskip("navi_amd.policy")

STRUCTS = {"navi_delta_rule": native.DeltaRule, "navi_delta_gradients": native.DeltaGradients,
           "navi_qk_norm_args": native.QkNorm}


def test_structures_match_the_header(tmp_path):
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "navi_policy.h"', "int main(void) {"]
    for c, py in STRUCTS.items():
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        lines += [f'printf("%zu\\n", offsetof({c}, {f}));' for f, _ in py._fields_]
    lines += [f'printf("%d\\n", {n});' for n in ("NAVI_POLICY_MAX_KEY_DIM", "NAVI_POLICY_MAX_NORM_DIM",
                                                  "NAVI_POLICY_CHUNK", "NAVI_POLICY_NORM_PARTIALS")]
    source = tmp_path / "layout.c"
    source.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-I", str(ROOT / "include" / "policy"), str(source), "-o", str(tmp_path / "layout")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for py in STRUCTS.values():
        want += [ctypes.sizeof(py)] + [getattr(py, f).offset for f, _ in py._fields_]
    want += [native.MAX_KEY_DIM, native.MAX_NORM_DIM, native.CHUNK, native.NORM_PARTIALS]
    assert got == want


def rule(**over):
    a = native.DeltaRule(dtype=native.F32, key_heads=2, value_heads=4, key_dim=16, value_dim=16, envs=2, steps=100, scale=1.0)
    for name in ("q", "k", "v", "g", "beta", "out", "matrices"):
        setattr(a, name, 4096)  # never read: every call here is refused before a launch
    for name, dim in (("q", 16), ("k", 16), ("v", 16)):
        setattr(a, name + "_stride", (ctypes.c_int64 * 3)(1 << 20, 4 * dim, dim))
    for name, value in over.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("over, words", [
    ({"dtype": 3}, "dtype must be"),
    ({"value_heads": 3}, "multiple of key_heads"),
    ({"key_heads": 0}, "multiple of key_heads"),
    ({"key_dim": 0}, "key_dim must be"),
    ({"key_dim": 129}, "key_dim must be"),
    ({"value_dim": 65537}, "value_dim must be"),
    ({"envs": -1}, "must not be negative"),
    ({"envs": 1 << 30}, "below 2^31"),
    ({"steps": 1 << 31}, "below 2^31"),
    ({"beta": None}, "must be non-null"),
])
def test_rule_refusals(over, words):
    for name in ("navi_delta_forward", "navi_delta_step"):
        code = getattr(native.lib(), name)(ctypes.byref(rule(**over)), None)
        assert code == native.NAVI_POLICY_E_ARG and words in native.last_error()
    with pytest.raises(RuntimeError, match=words.replace("^", r"\^")):
        native.check(code)


def test_rule_refusals_of_saved_arrays():
    lib = native.lib()
    assert lib.navi_delta_forward(ctypes.byref(rule(states=4096)), None) == native.NAVI_POLICY_E_ARG
    assert "saved together" in native.last_error()
    assert lib.navi_delta_step(ctypes.byref(rule(updates=4096)), None) == native.NAVI_POLICY_E_ARG
    d = native.DeltaGradients()
    assert lib.navi_delta_backward(ctypes.byref(rule()), ctypes.byref(d), None) == native.NAVI_POLICY_E_ARG
    for name in ("grad_out", "d_q", "d_k", "d_v", "d_g", "d_beta", "workspace"):
        setattr(d, name, 4096)
    assert lib.navi_delta_backward(ctypes.byref(rule()), ctypes.byref(d), None) == native.NAVI_POLICY_E_ARG
    assert "states and updates" in native.last_error()
    d.workspace = 4100
    assert lib.navi_delta_backward(ctypes.byref(rule(states=4096, updates=4096)), ctypes.byref(d), None) < 0
    assert "16-byte aligned" in native.last_error()


@pytest.mark.parametrize("name", ["q_stride", "v_stride"])
@pytest.mark.parametrize("step", [0, 15, 1 << 23, -64])
def test_steps_that_overlap_or_lie_far_apart_are_refused(name, step):
    a = rule(**{name: (ctypes.c_int64 * 3)(1 << 30, step, 16)})
    assert native.lib().navi_delta_forward(ctypes.byref(a), None) == native.NAVI_POLICY_E_ARG
    assert "overlap or lie too far apart" in native.last_error()
    wide = rule(value_heads=1 << 18, key_heads=1 << 18, value_dim=64, envs=1)
    assert native.lib().navi_delta_forward(ctypes.byref(wide), None) == native.NAVI_POLICY_E_ARG
    assert "value_heads * value_dim or" in native.last_error()


def test_workspace_sizes():
    lib = native.lib()
    # 8 sequences of 100 steps: one state gradient each, rows of 16, and key gradients per value head
    assert lib.navi_delta_workspace(ctypes.byref(rule())) == 4 * (8 * 256 + 8 * 100 * 16 + 2 * 8 * 100 * 16)
    assert lib.navi_delta_workspace(ctypes.byref(rule(key_heads=4))) == 4 * (8 * 256 + 8 * 100 * 16)
    assert lib.navi_delta_workspace(ctypes.byref(rule(key_dim=0))) < 0
    assert lib.navi_delta_forward(ctypes.byref(rule(envs=0)), None) == native.NAVI_POLICY_OK


@pytest.mark.parametrize("over, words", [
    ({"dtype": -1}, "dtype must be"),
    ({"norm": 2}, "norm must be"),
    ({"head_dim": 1025}, "head_dim must be"),
    ({"pairs": 33}, "pairs must be"),
    ({"pairs": 4}, "needs cos and sin"),
    ({"eps": -1.0}, "eps must not"),
    ({"envs": -2}, "must not be negative"),
    ({}, "must be non-null"),
])
def test_norm_refusals(over, words):
    a = native.QkNorm(head_dim=64, query_heads=1, key_heads=1, envs=1, steps=1)
    for name, value in over.items():
        setattr(a, name, value)
    assert native.lib().navi_qk_norm(ctypes.byref(a), None) == native.NAVI_POLICY_E_ARG
    assert words in native.last_error()


def test_clip_refusals():
    lib = native.lib()
    one = lambda t, v: (t * 1)(v)  # noqa: E731
    args = lambda **o: (1, one(ctypes.c_void_p, o.get("p", 4096)), one(ctypes.c_void_p, 4096),  # noqa: E731
                        one(ctypes.c_int64, o.get("n", 4)), one(ctypes.c_int32, o.get("t", 0)), o.get("m", 1.0), 1e-6,
                        o.get("norm", 4096), 4096, None)
    for over, words in (({"p": None}, "null"), ({"n": -1}, "invalid count"), ({"t": 5}, "must be float32"),
                        ({"m": -1.0}, "not be negative"), ({"m": float("nan")}, "not be negative"), ({"norm": None}, "non-null")):
        assert lib.navi_clip_grad_norm(*args(**over)) == native.NAVI_POLICY_E_ARG
        assert words in native.last_error()


def test_host_tensors_are_refused():
    q = torch.zeros(1, 2, 1, 8)
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        policy.gated_delta_rule(q, q, q, q[..., 0], q[..., 0])
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        policy.gated_delta_step(q[0], q[0], q[0], q[0, ..., 0], q[0, ..., 0], torch.zeros(2, 1, 8, 8))
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        policy.qk_norm(q, q)
    with pytest.raises(RuntimeError, match="CUDA"):
        policy.clip_grad_norm([q], 1.0)


def test_the_tests_own_definition():
    """Closed forms of the recurrence that the GPU tests compare with."""
    one = torch.ones(1, 4, 1, 1)
    gate = torch.full((1, 4, 1), -0.5)
    # beta = 1 with a unit key: the state becomes v whatever it was
    o, s = ref.rule(one, one, torch.arange(4.0).view(1, 4, 1, 1), gate, torch.ones(1, 4, 1), None, None, 2.0)
    assert torch.allclose(o.flatten(), 2.0 * torch.arange(4.0).double()) and float(s) == 3.0
    # beta = 0: it only decays, and a start clears it
    starts = torch.tensor([[False, False, True, False]])
    o, s = ref.rule(one, one, one, gate, torch.zeros(1, 4, 1), starts, torch.ones(1, 1, 1, 1), 1.0)
    assert torch.allclose(o.flatten(), torch.tensor([-0.5, -1.0, -torch.inf, -torch.inf]).exp().double())

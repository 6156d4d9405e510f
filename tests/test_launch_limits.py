"""A launch has fewer than 2^32 threads: calls of the selective scan, the gated delta rule, the raw tracer and the observation pass that would need more are
refused before anything runs (a larger grid is cut off without an error). Without a GPU: addresses are never read, and calls within the limit end at an argument that is left out."""

from __future__ import annotations

import ctypes
from pathlib import Path

import pytest

from navi_amd import _native as tracer
from navi_amd import _policy_native as native

from .test_block_boundary import PAGE, refused, scan, three
from .test_policy_boundary import rule

FAR = 1 << 44  # (inputs of that many environments end before the next)


def large(**over):
    places = {name: FAR * (i + 1) for i, name in enumerate(("x", "b", "c", "dt", "a"))}
    return scan(**{**places, "out": None, "scratch": 9 * PAGE, **over})


LIMITS = [  # the last that fits, the first that does not: workgroups of 64 columns of a head, rounded up to 8 envs
    (dict(envs=(1 << 22) - 8, heads=4, groups=4), dict(envs=1 << 22, heads=4, groups=4)),
    (dict(envs=(1 << 22) - 8, heads=4, groups=1, b_stride=three(160, 16, 16), c_stride=three(160, 16, 16)),
     dict(envs=(1 << 22) - 2, heads=4, groups=1, b_stride=three(160, 16, 16), c_stride=three(160, 16, 16))),
    (dict(envs=(1 << 20) - 8, heads=8, groups=8, head_dim=72, x_stride=three(5760, 576, 72)), dict(envs=1 << 20, heads=8, groups=8, head_dim=128)),
]


@pytest.mark.parametrize("fits, does_not", LIMITS[:2])
def test_scans(fits, does_not):
    lib = native.lib()
    refused(lib.navi_selective_scan(ctypes.byref(large(**fits)), None), "out must be")
    refused(lib.navi_selective_scan(ctypes.byref(large(**does_not)), None), "fewer than 2^32 threads")
    refused(lib.navi_selective_scan_backward(ctypes.byref(large(**does_not, grad_out=20 * FAR, grad_out_stride=three(320, 32, 8))), None),
            "fewer than 2^32 threads")


def test_scans_of_two_blocks_of_columns():
    fits, does_not = LIMITS[2]
    lib = native.lib()
    refused(lib.navi_selective_scan(ctypes.byref(large(**fits)), None), "out must be")
    refused(lib.navi_selective_scan(ctypes.byref(large(**does_not, x_stride=three(10240, 1024, 128))), None), "fewer than 2^32 threads")
    # backward also those of the state's columns
    wide = dict(envs=1 << 20, heads=8, groups=8, state_dim=65, b_stride=three(5200, 520, 65), c_stride=three(5200, 520, 65),
                x_stride=three(640, 64, 8), grad_out=20 * FAR, grad_out_stride=three(640, 64, 8))
    refused(lib.navi_selective_scan(ctypes.byref(large(**wide)), None), "out must be")
    refused(lib.navi_selective_scan_backward(ctypes.byref(large(**wide)), None), "fewer than 2^32 threads")


def test_gradients_of_many_chunks():
    """A workgroup a chunk of 64 tokens of a head."""
    lib = native.lib()
    size = dict(envs=1024, heads=16, groups=16, x_stride=three(1 << 23, 128, 8), b_stride=three(1 << 24, 256, 16),
                c_stride=three(1 << 24, 256, 16), grad_out=20 * FAR, grad_out_stride=three(1 << 23, 128, 8))
    refused(lib.navi_selective_scan(ctypes.byref(large(**size, steps=65536)), None), "out must be")
    refused(lib.navi_selective_scan_backward(ctypes.byref(large(**size, steps=65536)), None), "fewer than 2^32 threads")
    refused(lib.navi_selective_scan_backward(ctypes.byref(large(**size, steps=65472)), None), "must be non-null")


def test_single_tokens():
    """Four waves a workgroup, a wave 32 columns of a head (8 where rows are not multiples of four)."""
    lib = native.lib()
    one = dict(steps=1, heads=16, groups=16, x_stride=three(128, 128, 8), b_stride=three(256, 256, 16), c_stride=three(256, 256, 16),
               dt_stride=three(16, 16, 1), initial_state=30 * FAR, final_state=30 * FAR, out=40 * FAR)
    refused(lib.navi_selective_step(ctypes.byref(large(**{**one, "envs": 1 << 22})), None), "fewer than 2^32 threads")


@pytest.mark.parametrize("fits, does_not", [
    (dict(envs=(1 << 22) - 8, steps=1), dict(envs=1 << 22, steps=1)),
    (dict(envs=(1 << 20) - 8, steps=1, value_dim=256), dict(envs=1 << 20, steps=1, value_dim=256)),
    (dict(envs=1024, steps=64 * 4095), dict(envs=1024, steps=64 * 4096)),
    (dict(envs=(1 << 21) - 8, steps=1, key_dim=100, value_dim=129), dict(envs=1 << 21, steps=1, key_dim=100, value_dim=129)),  # (512 threads)
])
def test_delta_rules(fits, does_not):
    lib = native.lib()
    strides = dict(q_stride=three(1 << 40, 1 << 10, 128), k_stride=three(1 << 40, 1 << 10, 128), v_stride=three(1 << 40, 1 << 10, 256))
    if "value_dim" not in fits:
        assert lib.navi_delta_forward(ctypes.byref(rule(**strides, **fits, states=4096)), None) == native.NAVI_POLICY_E_ARG
        assert "2^32" not in native.last_error()
    refused(lib.navi_delta_forward(ctypes.byref(rule(**strides, **does_not)), None), "fewer than 2^32 threads")
    gradients = native.DeltaGradients()
    refused(lib.navi_delta_backward(ctypes.byref(rule(**strides, **does_not)), ctypes.byref(gradients), None), "fewer than 2^32 threads")


def test_gradients_of_delta_rules():
    """512 threads a chunk, 256 for float16 and keys of up to 64."""
    lib = native.lib()
    strides = dict(q_stride=three(1 << 40, 1 << 10, 128), k_stride=three(1 << 40, 1 << 10, 128), v_stride=three(1 << 40, 1 << 10, 256))
    gradients = native.DeltaGradients()
    for dtype, key_dim, chunks in ((native.F32, 64, 2047), (native.BF16, 64, 2047), (native.F16, 64, 4095), (native.F16, 65, 2047)):
        size = dict(envs=1024, dtype=dtype, key_dim=key_dim)
        refused(lib.navi_delta_backward(ctypes.byref(rule(**strides, **size, steps=64 * chunks)), ctypes.byref(gradients), None), "must be non-null")
        refused(lib.navi_delta_backward(ctypes.byref(rule(**strides, **size, steps=64 * chunks + 1)), ctypes.byref(gradients), None),
                "fewer than 2^32 threads")


def test_single_tokens_of_delta_rules():
    assert native.lib().navi_delta_step(ctypes.byref(rule(envs=1 << 24, steps=1, final_state=1 << 50, out=1 << 55)), None) == native.NAVI_POLICY_E_ARG
    assert "fewer than 2^32 threads" in native.last_error()


def test_heads_are_those_of_the_header():
    header = (Path(__file__).resolve().parents[1] / "include" / "policy" / "navi_policy.h").read_text()
    assert f"#define NAVI_POLICY_MAX_HEADS {native.MAX_HEADS}\n" in header


def test_rays_and_observations():
    """The raw tracer takes a ray a thread, the observation pass a workgroup of 512 an environment."""
    lib, f3 = tracer.lib(), tracer.float3
    for rays in ((1 << 32) - 255, 1 << 32, 1 << 36):
        code = lib.navi_cast_rays(4096, 1, 4096, 4096, 4096, 4096, rays, 4, 1.0, f3([0, 0, 0]), f3([1, 1, 1]), 1, 0.01, None, None, None)
        assert code == tracer.NAVI_E_ARG and "too many rays" in tracer.last_error()
    for envs in (1 << 23, (1 << 31) - 1):
        seen = tracer.Observation(distances=4096, semantics=4096, n_envs=envs, azimuth_bins=4, elevation_bins=2, max_distance=1.0, obs=1 << 50)
        assert lib.navi_observe(ctypes.byref(seen), None, None) == tracer.NAVI_E_ARG and "too many envs" in tracer.last_error()

"""The boundary of a block's operators (convolution, selective scan, norms, orthogonalised updates) without a
GPU: the C ABI's structures, sizes and argument checks, and what the Python layer refuses before any launch."""

from __future__ import annotations

import ctypes
import math
import subprocess
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]
native = pytest.importorskip("navi_amd._policy_native")
policy = pytest.importorskip("navi_amd.policy")

STRUCTS = {"navi_causal_conv_args": native.CausalConv, "navi_block_norm_args": native.BlockNorm,
           "navi_selective_scan_args": native.SelectiveScan, "navi_orthogonalize_matrix": native.OrthogonalizeMatrix}
CONSTANTS = {"NAVI_POLICY_MAX_TAPS": native.MAX_TAPS, "NAVI_POLICY_MAX_BLOCK_WIDTH": native.MAX_BLOCK_WIDTH,
             "NAVI_POLICY_MAX_STATE_DIM": native.MAX_STATE_DIM, "NAVI_POLICY_NONE": native.ACT_NONE,
             "NAVI_POLICY_SILU": native.ACT_SILU}
PAGE = 1 << 20  # addresses below are never read: every call here is refused, or empty, before a launch


def test_structures_match_the_header(tmp_path):
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "navi_policy.h"', "int main(void) {"]
    for c, py in STRUCTS.items():
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        lines += [f'printf("%zu\\n", offsetof({c}, {f.rstrip("_")}));' for f, _ in py._fields_]
    lines += [f'printf("%d\\n", {n});' for n in CONSTANTS]
    source = tmp_path / "layout.c"
    source.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-I", str(ROOT / "include" / "policy"), str(source), "-o", str(tmp_path / "layout")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for py in STRUCTS.values():
        want += [ctypes.sizeof(py)] + [getattr(py, f).offset for f, _ in py._fields_]
    assert got == want + list(CONSTANTS.values())


def two(*v):
    return (ctypes.c_int64 * 2)(*v)


def three(*v):
    return (ctypes.c_int64 * 3)(*v)


def filled(a, over):
    for name, value in over.items():
        setattr(a, name, value)
    return a


def conv(**over):
    a = native.CausalConv(dtype=native.F32, channels=16, taps=4, envs=2, steps=10, x=PAGE, x_stride=two(160, 16),
                          weight=2 * PAGE, out=3 * PAGE)
    return filled(a, over)


def block(**over):
    a = native.BlockNorm(dtype=native.BF16, stream_dtype=native.F32, width=64, eps=1e-6, envs=2, steps=10, y=PAGE,
                         residual=2 * PAGE, y_stride=two(640, 64), residual_stride=two(640, 64), stream=3 * PAGE,
                         normed=4 * PAGE)
    return filled(a, over)


def scan(**over):
    a = native.SelectiveScan(dtype=native.F32, heads=4, groups=2, state_dim=16, head_dim=8, envs=2, steps=10, x=PAGE,
                             b=2 * PAGE, c=3 * PAGE, x_stride=three(320, 32, 8), b_stride=three(320, 32, 16),
                             c_stride=three(320, 32, 16), dt=4 * PAGE, dt_stride=three(40, 4, 1), a=5 * PAGE, out=6 * PAGE)
    return filled(a, over)


def refused(code, words):
    assert code == native.NAVI_POLICY_E_ARG and words in native.last_error(), (code, native.last_error())


@pytest.mark.parametrize("over, words", [
    ({"dtype": 3}, "dtype must be"),
    ({"taps": 1}, "taps must be"),
    ({"taps": 5}, "taps must be"),
    ({"channels": 0}, "channels must be"),
    ({"channels": 65537}, "channels must be"),
    ({"activation": 2}, "activation must be"),
    ({"envs": -1}, "must not be negative"),
    ({"steps": 1 << 31}, "below 2^31"),
    ({"x_stride": two(-160, 16)}, "strides must not be negative"),
    ({"x": None}, "x and weight must be"),
    ({"weight": None}, "x and weight must be"),
    ({"weight": 2 * PAGE + 2}, "aligned to their elements"),
    ({"x": PAGE + 2}, "aligned to their elements"),
    ({"x": 4 * PAGE, "x_stride": two(1 << 40, 1 << 30)}, "within 2 GiB"),
])
def test_conv_refusals(over, words):
    refused(native.lib().navi_causal_conv(ctypes.byref(conv(**over)), None), words)
    backward = conv(grad_out=7 * PAGE, grad_out_stride=two(160, 16), d_x=8 * PAGE, **over)
    refused(native.lib().navi_causal_conv_backward(ctypes.byref(backward), None), words)


def test_conv_refusals_of_outputs():
    lib = native.lib()
    refused(lib.navi_causal_conv(None, None), "args must be")
    refused(lib.navi_causal_conv(ctypes.byref(conv(out=None)), None), "out must be")
    refused(lib.navi_causal_conv_backward(ctypes.byref(conv()), None), "grad_out and d_x")
    refused(lib.navi_causal_conv_backward(ctypes.byref(conv(steps=0)), None), "at least one step")
    refused(lib.navi_causal_conv_backward(ctypes.byref(conv(grad_out=7 * PAGE, d_x=8 * PAGE, d_bias=9 * PAGE)), None), "workspace")


@pytest.mark.parametrize("over", [
    {"out": PAGE},                                # the input of a whole rollout
    {"out": 2 * PAGE - 64},                       # the weight
    {"out": PAGE + 4 * 319},                      # the input's last number
    {"window_out": PAGE}, {"window_out": 3 * PAGE},
    {"window": 9 * PAGE, "window_out": 9 * PAGE + 4},  # the window, shifted
    {"bias": 9 * PAGE, "window_out": 9 * PAGE + 60},
    {"starts": 9 * PAGE, "starts_stride": two(10, 1), "out": 9 * PAGE + 16},
])
def test_conv_outputs_that_share_memory(over):
    refused(native.lib().navi_causal_conv(ctypes.byref(conv(**over)), None), "shares memory")


@pytest.mark.parametrize("over, words", [
    ({"dtype": -1}, "dtype must be"),
    ({"stream_dtype": native.F16}, "stream_dtype must be"),
    ({"dtype": native.F32, "stream_dtype": native.BF16}, "stream_dtype must be"),
    ({"width": 0}, "width must be"),
    ({"width": 8193}, "width must be"),
    ({"eps": -1.0}, "eps must not"),
    ({"eps": math.nan}, "eps must not"),
    ({"envs": -1}, "must not be negative"),
    ({"envs": 1 << 30}, "below 2^31"),
    ({"y": None}, "y and residual must be"),
    ({"residual": 2 * PAGE + 2}, "aligned to their elements"),
    ({"gate": 9 * PAGE + 1}, "aligned to their elements"),
    ({"scale": 9 * PAGE + 2}, "aligned to their elements"),
])
def test_block_refusals(over, words):
    refused(native.lib().navi_block_norm(ctypes.byref(block(**over)), None), words)
    backward = block(d_y=7 * PAGE, d_residual=8 * PAGE, **over)
    assert native.lib().navi_block_norm_backward(ctypes.byref(backward), None) == native.NAVI_POLICY_E_ARG


def test_block_refusals_of_outputs():
    lib = native.lib()
    refused(lib.navi_block_norm(None, None), "args must be")
    refused(lib.navi_block_norm(ctypes.byref(block(stream=None)), None), "stream and normed")
    refused(lib.navi_block_norm_backward(ctypes.byref(block(steps=0)), None), "at least one row")
    refused(lib.navi_block_norm_backward(ctypes.byref(block(d_y=7 * PAGE)), None), "d_y and d_residual")
    refused(lib.navi_block_norm_backward(ctypes.byref(block(d_y=7 * PAGE, d_residual=8 * PAGE, d_scale=9 * PAGE)), None), "workspace")
    for over in ({"stream": PAGE}, {"normed": 2 * PAGE}, {"stream": 4 * PAGE + 64}, {"normed": 9 * PAGE, "gate": 9 * PAGE},
                 {"stream": 2 * PAGE + 16, "residual_stride": two(640, 64)}):
        refused(lib.navi_block_norm(ctypes.byref(block(**over)), None), "shares memory")


SCAN = [
    ({"dtype": 3}, "dtype must be"),
    ({"groups": 3}, "multiple of groups"),
    ({"heads": 0}, "multiple of groups"),
    ({"state_dim": 129}, "must be in [1, 128]"),
    ({"head_dim": 0}, "must be in [1, 128]"),
    ({"heads": 16386}, "at most 16384"),
    ({"envs": -1}, "must not be negative"),
    ({"envs": 1 << 29}, "below 2^31"),
    ({"steps": 1 << 31}, "below 2^31"),
    ({"x": None}, "must be non-null"),
    ({"a": None}, "must be non-null"),
    ({"dt": 4 * PAGE + 2}, "aligned to their elements"),
    ({"b": 2 * PAGE + 1}, "aligned to their elements"),
]


@pytest.mark.parametrize("over, words", SCAN)
def test_scan_refusals(over, words):
    lib = native.lib()
    refused(lib.navi_selective_scan(ctypes.byref(scan(scratch=9 * PAGE, **over)), None), words)
    one = dict(steps=1, initial_state=8 * PAGE, final_state=8 * PAGE)
    one.update(over)
    refused(lib.navi_selective_step(ctypes.byref(scan(**one)), None), words)
    backward = scan(grad_out=7 * PAGE, grad_out_stride=three(320, 32, 8), d_x=10 * PAGE, d_b=11 * PAGE, d_c=12 * PAGE,
                    d_dt=13 * PAGE, workspace=16 * PAGE, **over)
    refused(lib.navi_selective_scan_backward(ctypes.byref(backward), None), words)


@pytest.mark.parametrize("name", ["x_stride", "b_stride", "c_stride"])
@pytest.mark.parametrize("step", [0, 3, 1 << 24, -64])
def test_scans_over_steps_that_overlap_or_lie_far_apart(name, step):
    a = scan(steps=1000, scratch=9 * PAGE, **{name: three(1 << 40, step, 16)})
    refused(native.lib().navi_selective_scan(ctypes.byref(a), None), "overlap or lie too far apart")


def test_scan_refusals_of_outputs():
    lib = native.lib()
    refused(lib.navi_selective_scan(None, None), "args must be")
    refused(lib.navi_selective_scan(ctypes.byref(scan(out=None, scratch=9 * PAGE)), None), "out must be")
    refused(lib.navi_selective_scan_backward(ctypes.byref(scan(grad_out_stride=three(320, 32, 8))), None), "must be non-null")
    refused(lib.navi_selective_scan_backward(ctypes.byref(scan(steps=0)), None), "at least one token")
    backward = scan(grad_out=7 * PAGE, grad_out_stride=three(320, 32, 8), d_x=10 * PAGE, d_b=11 * PAGE, d_c=12 * PAGE,
                    d_dt=13 * PAGE, workspace=16 * PAGE + 4)
    refused(lib.navi_selective_scan_backward(ctypes.byref(backward), None), "16-byte aligned")
    # a scan long enough to be cut into parts: their states go to the scratch
    long = scan(envs=1, steps=100000)
    assert lib.navi_selective_scan_scratch(ctypes.byref(long)) > 0
    refused(lib.navi_selective_scan(ctypes.byref(long), None), "scratch must be")
    refused(lib.navi_selective_scan(ctypes.byref(scan(envs=1, steps=100000, out=200 * PAGE, scratch=400 * PAGE + 4)), None),
            "scratch must be")


@pytest.mark.parametrize("over", [
    {"out": PAGE}, {"out": 2 * PAGE + 64}, {"out": 3 * PAGE}, {"out": 4 * PAGE}, {"out": 5 * PAGE},
    {"final_state": 6 * PAGE}, {"final_state": 3 * PAGE},
    {"initial_state": 9 * PAGE, "final_state": 9 * PAGE + 16},
    {"d": 9 * PAGE, "final_state": 9 * PAGE}, {"dt_bias": 9 * PAGE, "out": 9 * PAGE - 16},
    {"starts": 9 * PAGE, "starts_stride": two(10, 1), "out": 9 * PAGE},
])
def test_scan_outputs_that_share_memory(over):
    refused(native.lib().navi_selective_scan(ctypes.byref(scan(scratch=20 * PAGE, **over)), None), "shares memory")


def test_one_token_where_memory_is_shared():
    lib = native.lib()
    one = dict(steps=1, initial_state=8 * PAGE, final_state=8 * PAGE)
    for over in ({"out": 2 * PAGE}, {"out": 8 * PAGE + 64}, {"out": PAGE + 4}, {"final_state": 8 * PAGE + 64},
                 {"initial_state": PAGE, "final_state": PAGE}):
        refused(lib.navi_selective_step(ctypes.byref(scan(**{**one, **over})), None), "shares memory")


def matrices(*rows):
    made = [dict(from_=PAGE * (2 * i + 1), to=PAGE * (2 * i + 2), rows=16, cols=32, from_stride=two(32, 1),
                 to_stride=two(32, 1)) | row for i, row in enumerate(rows)]
    return len(rows), (native.OrthogonalizeMatrix * max(1, len(rows)))(*[native.OrthogonalizeMatrix(**m) for m in made])


def orthogonalize(array, steps=5, factors=(3.4445, -4.775, 2.0315), eps=1e-7, workspace=64 * PAGE):
    return native.lib().navi_orthogonalize(*array, steps, *factors, eps, workspace, None)


@pytest.mark.parametrize("row, words", [
    ({"rows": (1 << 20) + 1}, "at most 2^20"),
    ({"rows": 1 << 20, "cols": 1 << 11}, "2^31 numbers"),
    ({"cols": -1}, "at most 2^20"),
    ({"from_dtype": 3}, "must be float32, bfloat16 or float16"),
    ({"to_dtype": -1}, "must be float32, bfloat16 or float16"),
    ({"from_": None}, "is null"),
    ({"to": PAGE * 2 + 2}, "aligned to its elements"),
    ({"from_stride": two(64, 2)}, "contiguous along"),
    ({"to": PAGE + 64}, "share memory"),
])
def test_orthogonalize_refusals(row, words):
    refused(orthogonalize(matrices({}, row)), words)


def test_orthogonalize_refusals_of_what_is_not_a_matrix():
    refused(native.lib().navi_orthogonalize(1, None, 5, 1.0, 1.0, 1.0, 0.0, 64 * PAGE, None), "must be non-null")
    refused(orthogonalize((-1, None)), "must be non-null")
    refused(orthogonalize(matrices({}), steps=0), "steps must be")
    refused(orthogonalize(matrices({}), steps=101), "steps must be")
    refused(orthogonalize(matrices({}), eps=-1.0), "eps must not")
    refused(orthogonalize(matrices({}), factors=(math.inf, 1.0, 1.0)), "must be finite")
    refused(orthogonalize(matrices({}), workspace=None), "workspace must be")
    refused(orthogonalize(matrices({}), workspace=64 * PAGE + 128), "workspace must be")
    refused(orthogonalize(matrices({}, {"to": PAGE * 2})), "that are written share memory")
    refused(orthogonalize(matrices({}, {"to": PAGE})), "share memory")  # (another's input, the same place)
    assert orthogonalize((0, None), workspace=None) == native.NAVI_POLICY_OK


def test_workspace_sizes():
    lib = native.lib()
    assert lib.navi_causal_conv_workspace(ctypes.byref(conv())) > 0
    assert lib.navi_block_norm_workspace(ctypes.byref(block())) > 0
    assert lib.navi_selective_scan_workspace(ctypes.byref(scan())) > 0
    assert lib.navi_orthogonalize_workspace(*matrices({}, {})) > 0
    assert lib.navi_selective_scan_scratch(ctypes.byref(scan(envs=1024, steps=16))) == 0
    for name, bad in (("navi_causal_conv_workspace", conv(taps=9)), ("navi_block_norm_workspace", block(width=0)),
                      ("navi_selective_scan_workspace", scan(groups=3)), ("navi_selective_scan_scratch", scan(groups=3))):
        assert getattr(lib, name)(ctypes.byref(bad)) < 0
    assert lib.navi_orthogonalize_workspace(*matrices({"rows": -1})) < 0


def test_calls_of_no_rows():
    lib = native.lib()
    assert lib.navi_causal_conv(ctypes.byref(conv(envs=0)), None) == native.NAVI_POLICY_OK
    assert lib.navi_block_norm(ctypes.byref(block(envs=0)), None) == native.NAVI_POLICY_OK
    assert lib.navi_block_norm(ctypes.byref(block(steps=0)), None) == native.NAVI_POLICY_OK
    assert lib.navi_selective_scan(ctypes.byref(scan(envs=0, scratch=9 * PAGE)), None) == native.NAVI_POLICY_OK
    assert lib.navi_selective_step(ctypes.byref(scan(envs=0, steps=1)), None) == native.NAVI_POLICY_OK


def test_host_tensors_are_refused():
    x, b, h = torch.zeros(1, 2, 1, 8), torch.zeros(1, 2, 1, 4), torch.zeros(1)
    with pytest.raises(RuntimeError, match="x must be a CUDA tensor"):
        policy.selective_scan(x, x[..., 0], h, b, b)
    with pytest.raises(RuntimeError, match="x must be a CUDA tensor"):
        policy.selective_scan_step(x[0], x[0, ..., 0], h, b[0], b[0], torch.zeros(2, 1, 4, 8))
    with pytest.raises(RuntimeError, match="x must be a CUDA tensor"):
        policy.causal_conv(x[0], torch.zeros(8, 4))
    with pytest.raises(RuntimeError, match="x must be a CUDA tensor"):
        policy.causal_conv_step(x[0, 0], torch.zeros(8, 4), torch.zeros(1, 3, 8))
    with pytest.raises(RuntimeError, match="y must be a CUDA tensor"):
        policy.block_norm(x[0], x[0])
    with pytest.raises(RuntimeError, match="CUDA"):
        policy.orthogonalize([x[0, 0]])


def test_what_is_no_tensor_is_refused():
    with pytest.raises(RuntimeError, match="x must be a CUDA tensor"):
        policy.selective_scan_step(None, 1, "a", [], {}, ())
    with pytest.raises(RuntimeError, match="x must be a CUDA tensor"):
        policy.causal_conv_step(1.0, None, None, activation=object())
    with pytest.raises(RuntimeError, match="y must be a CUDA tensor"):
        policy.block_norm(None, None)
    for eps in (-1.0, math.nan, math.inf):
        with pytest.raises(RuntimeError):
            policy.block_norm(torch.zeros(1, 1, 4), torch.zeros(1, 1, 4), eps=eps)


def test_the_extension_leaves_what_it_does_not_take():
    """Host tensors, other types, a wrong number of arguments: None, and nothing done."""
    calls, x = native.calls, torch.zeros(2, 1, 8)
    assert calls.selective_step(x, x, x, x, x, x, None, None, None, None) is None
    assert calls.selective_step() is None
    assert calls.conv_step(x, x, x, None, None, 0, None) is None
    assert calls.conv_step(x, x, x, None, None, None, None) is None
    assert calls.block_norm(x, x, None, None, None, None, 1e-6) is None
    assert calls.block_norm(x, x, None, None, None, None, "1") is None
    assert calls.selective_scan(x, x, x, x, x, None, None, None, None, False, 4) is None
    assert calls.selective_scan(x) is None
    assert calls.causal_conv(x, x, None, None, None, 1, False) is None
    assert calls.causal_conv(x, x, None, None, None, None, False) is None
    sparse = torch.eye(4).to_sparse()
    assert calls.block_norm(sparse, sparse, None, None, None, None, 1e-6) is None
    with pytest.raises(TypeError):
        calls.bind(1)

"""ctypes binding of ``libnavi_policy.so`` (the C ABI declared in ``include/policy/navi_policy.h``),
and ``calls``, the extension that makes calls of some of it in one step (``csrc/policy/calls.cpp``).

Importing this module loads the HIP library and raises ``ImportError`` when it has not been
built; there is no fallback. Where the extension is missing, or made for another PyTorch, its operators
(selective scan, convolution, block norms) raise, and all others work.
"""

from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import os
import struct
from pathlib import Path

import torch  # noqa: F401  (the extension's libraries)

LIB_DIR = Path(__file__).resolve().parent / "_lib"
LIB_PATH = Path(os.environ.get("NAVI_POLICY_LIB", LIB_DIR / "libnavi_policy.so"))
CALLS_PATH = LIB_DIR / "_policy_calls.so"

NAVI_POLICY_OK = 0
NAVI_POLICY_E_ARG = -1
NAVI_POLICY_E_LAUNCH = -2
F32, BF16, F16 = 0, 1, 2
MAX_KEY_DIM, MAX_NORM_DIM, CHUNK, CHUNK_MATRICES = 128, 1024, 64, 5248
NORM_RMS, NORM_L2 = 0, 1
NORM_PARTIALS = 2048
MAX_TAPS, MAX_BLOCK_WIDTH, MAX_STATE_DIM, MAX_HEADS = 4, 8192, 128, 16384
ACT_NONE, ACT_SILU = 0, 1

_BUILD = "build it with `python -c 'import __graft_entry__ as g; g.build()'` (or `make -C navi_amd/csrc/policy`)."

if not LIB_PATH.exists():
    raise ImportError(f"{LIB_PATH.name} not found at {LIB_PATH}; {_BUILD}")
_lib = ctypes.CDLL(str(LIB_PATH))

_vp, _i32, _i64, _f32 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float
_three, _two = ctypes.c_int64 * 3, ctypes.c_int64 * 2


class DeltaRule(ctypes.Structure):
    """navi_delta_rule (include/policy/navi_policy.h)."""

    _fields_ = [("dtype", _i32), ("key_heads", _i32), ("value_heads", _i32), ("key_dim", _i32), ("value_dim", _i32),
                ("envs", _i64), ("steps", _i64), ("scale", _f32), ("q", _vp), ("k", _vp), ("v", _vp),
                ("q_stride", _three), ("k_stride", _three), ("v_stride", _three), ("g", _vp), ("beta", _vp),
                ("g_stride", _three), ("beta_stride", _three), ("starts", _vp), ("starts_stride", _two),
                ("initial_state", _vp), ("out", _vp), ("final_state", _vp), ("matrices", _vp), ("scratch", _vp),
                ("states", _vp), ("updates", _vp)]


class DeltaGradients(ctypes.Structure):
    """navi_delta_gradients (include/policy/navi_policy.h)."""

    _fields_ = [("grad_out", _vp), ("grad_out_stride", _three), ("grad_final_state", _vp), ("d_q", _vp),
                ("d_k", _vp), ("d_v", _vp), ("d_g", _vp), ("d_beta", _vp), ("d_initial_state", _vp),
                ("workspace", _vp)]


class QkNorm(ctypes.Structure):
    """navi_qk_norm_args (include/policy/navi_policy.h)."""

    _fields_ = [("dtype", _i32), ("norm", _i32), ("query_heads", _i32), ("key_heads", _i32), ("head_dim", _i32),
                ("pairs", _i32), ("interleaved", _i32), ("positions_wide", _i32), ("envs", _i64), ("steps", _i64),
                ("eps", _f32), ("q", _vp), ("k", _vp), ("q_stride", _three), ("k_stride", _three),
                ("q_weight", _vp), ("k_weight", _vp), ("positions", _vp), ("positions_stride", _two), ("cos", _vp),
                ("sin", _vp), ("positions_end", _i64), ("q_out", _vp), ("k_out", _vp), ("grad_q", _vp),
                ("grad_k", _vp), ("grad_q_stride", _three), ("grad_k_stride", _three), ("d_q", _vp), ("d_k", _vp),
                ("d_q_weight", _vp), ("d_k_weight", _vp), ("partial", _vp)]


class CausalConv(ctypes.Structure):
    """navi_causal_conv_args (include/policy/navi_policy.h)."""

    _fields_ = [("dtype", _i32), ("channels", _i32), ("taps", _i32), ("activation", _i32), ("envs", _i64), ("steps", _i64),
                ("x", _vp), ("x_stride", _two), ("weight", _vp), ("bias", _vp), ("starts", _vp), ("starts_stride", _two),
                ("window", _vp), ("out", _vp), ("window_out", _vp), ("grad_out", _vp), ("grad_out_stride", _two),
                ("grad_window", _vp), ("d_x", _vp), ("d_weight", _vp), ("d_bias", _vp), ("d_window", _vp), ("partial", _vp)]


class BlockNorm(ctypes.Structure):
    """navi_block_norm_args (include/policy/navi_policy.h)."""

    _fields_ = [("dtype", _i32), ("stream_dtype", _i32), ("width", _i32), ("eps", _f32), ("envs", _i64), ("steps", _i64),
                ("y", _vp), ("residual", _vp), ("gate", _vp), ("y_stride", _two), ("residual_stride", _two),
                ("gate_stride", _two), ("scale", _vp), ("post_weight", _vp), ("pre_weight", _vp), ("stream", _vp),
                ("normed", _vp), ("grad_stream", _vp), ("grad_normed", _vp), ("grad_stream_stride", _two),
                ("grad_normed_stride", _two), ("d_y", _vp), ("d_residual", _vp), ("d_gate", _vp), ("d_scale", _vp),
                ("d_post_weight", _vp), ("d_pre_weight", _vp), ("partial", _vp)]


class SelectiveScan(ctypes.Structure):
    """navi_selective_scan_args (include/policy/navi_policy.h)."""

    _fields_ = [("dtype", _i32), ("heads", _i32), ("groups", _i32), ("state_dim", _i32), ("head_dim", _i32), ("envs", _i64),
                ("steps", _i64), ("x", _vp), ("b", _vp), ("c", _vp), ("x_stride", _three), ("b_stride", _three),
                ("c_stride", _three), ("dt", _vp), ("dt_stride", _three), ("a", _vp), ("d", _vp), ("dt_bias", _vp),
                ("starts", _vp), ("starts_stride", _two), ("initial_state", _vp), ("out", _vp), ("final_state", _vp),
                ("scratch", _vp), ("grad_out", _vp), ("grad_out_stride", _three), ("grad_final_state", _vp), ("d_x", _vp),
                ("d_b", _vp), ("d_c", _vp), ("d_dt", _vp), ("d_a", _vp), ("d_d", _vp), ("d_dt_bias", _vp),
                ("d_initial_state", _vp), ("workspace", _vp)]


class OrthogonalizeMatrix(ctypes.Structure):
    """navi_orthogonalize_matrix (include/policy/navi_policy.h)."""

    _fields_ = [("from_", _vp), ("to", _vp), ("rows", _i64), ("cols", _i64), ("from_stride", _two), ("to_stride", _two),
                ("from_dtype", _i32), ("to_dtype", _i32)]


def _packer(structure) -> struct.Struct:
    """The structure's fields in order as a packer of plain numbers (an array's one by one): a
    call's arguments in one step, a fifth of the time that setting the fields takes."""
    codes = {_i32: "i", _i64: "q", _f32: "f", _vp: "P", _three: "3q", _two: "2q"}
    packer = struct.Struct("@" + "".join(codes[kind] for _, kind in structure._fields_) + "0q")
    assert packer.size == ctypes.sizeof(structure)
    return packer


PACK_RULE, PACK_GRADIENTS, PACK_NORM = (_packer(s).pack for s in (DeltaRule, DeltaGradients, QkNorm))
PACK_CONV, PACK_SCAN = (_packer(s).pack for s in (CausalConv, SelectiveScan))
PACK_MATRIX = _packer(OrthogonalizeMatrix).pack

_lib.navi_policy_last_error.restype = ctypes.c_char_p
_lib.navi_policy_last_error.argtypes = []
# (structures as bytes or by reference)
for _name in ("navi_delta_forward", "navi_delta_step", "navi_qk_norm", "navi_qk_norm_backward",
              "navi_causal_conv", "navi_causal_conv_backward", "navi_block_norm", "navi_block_norm_backward",
              "navi_selective_scan", "navi_selective_scan_backward", "navi_selective_step"):
    getattr(_lib, _name).restype = ctypes.c_int
    getattr(_lib, _name).argtypes = [_vp, _vp]
for _name in ("navi_delta_scratch", "navi_delta_workspace", "navi_qk_norm_workspace", "navi_causal_conv_workspace",
              "navi_block_norm_workspace", "navi_selective_scan_scratch", "navi_selective_scan_workspace"):
    getattr(_lib, _name).restype = _i64
    getattr(_lib, _name).argtypes = [_vp]
_lib.navi_delta_backward.restype = ctypes.c_int
_lib.navi_delta_backward.argtypes = [_vp, _vp, _vp]
_lib.navi_orthogonalize.restype = ctypes.c_int
_lib.navi_orthogonalize.argtypes = [_i32, _vp, _i32, _f32, _f32, _f32, _f32, _vp, _vp]
_lib.navi_orthogonalize_workspace.restype = _i64
_lib.navi_orthogonalize_workspace.argtypes = [_i32, _vp]
_lib.navi_clip_grad_norm.restype = ctypes.c_int
_lib.navi_clip_grad_norm.argtypes = [_i32, _vp, _vp, _vp, _vp, _f32, _f32, _vp, _vp, _vp]


class _NoCalls:
    """In the extension's place where there is none: whoever asks for one of its calls is told why."""

    def __init__(self, why: str) -> None:
        self._why = why

    def __getattr__(self, name: str):
        raise RuntimeError(self._why)


def _load_calls():
    if not CALLS_PATH.exists():
        return _NoCalls(f"{CALLS_PATH.name} not found at {CALLS_PATH}; {_BUILD}")
    loader = importlib.machinery.ExtensionFileLoader("_policy_calls", str(CALLS_PATH))
    try:
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_policy_calls", loader))
    except ImportError as e:  # (made for another PyTorch or Python)
        return _NoCalls(f"{CALLS_PATH.name} does not load ({e}); {_BUILD}")
    module.bind(*[ctypes.cast(getattr(_lib, name), _vp).value
                  for name in ("navi_selective_step", "navi_selective_scan", "navi_selective_scan_backward",
                               "navi_selective_scan_scratch", "navi_selective_scan_workspace", "navi_causal_conv",
                               "navi_causal_conv_backward", "navi_causal_conv_workspace", "navi_block_norm",
                               "navi_block_norm_backward", "navi_block_norm_workspace", "navi_policy_last_error")])
    return module


calls = _load_calls()


def lib() -> ctypes.CDLL:
    return _lib


def last_error() -> str:
    return _lib.navi_policy_last_error().decode(errors="replace")


def check(code: int) -> int:
    """Raise ``RuntimeError`` for a failed call; a size (a code >= 0) is returned."""
    if code < 0:
        raise RuntimeError(last_error() or f"navi_policy call failed with code {code}")
    return code

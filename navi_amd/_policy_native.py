"""ctypes binding of ``libnavi_policy.so`` (the C ABI declared in ``include/policy/navi_policy.h``).

Importing this module loads the HIP library and raises ``ImportError`` when it has not been
built; there is no fallback.
"""

from __future__ import annotations

import ctypes
import os
import struct
from pathlib import Path

LIB_DIR = Path(__file__).resolve().parent / "_lib"
LIB_PATH = Path(os.environ.get("NAVI_POLICY_LIB", LIB_DIR / "libnavi_policy.so"))

NAVI_POLICY_OK = 0
NAVI_POLICY_E_ARG = -1
NAVI_POLICY_E_LAUNCH = -2
F32, BF16, F16 = 0, 1, 2
MAX_KEY_DIM, MAX_NORM_DIM, CHUNK, CHUNK_MATRICES = 128, 1024, 64, 5248
NORM_RMS, NORM_L2 = 0, 1
NORM_PARTIALS = 2048

if not LIB_PATH.exists():
    raise ImportError(
        f"libnavi_policy.so not found at {LIB_PATH}; build it with "
        "`python -c 'import __graft_entry__ as g; g.build()'` (or `make -C navi_amd/csrc/policy`)."
    )
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


def _packer(structure) -> struct.Struct:
    """The structure's fields in order as a packer of plain numbers (an array's one by one): a
    call's arguments in one step, a fifth of the time that setting the fields takes."""
    codes = {_i32: "i", _i64: "q", _f32: "f", _vp: "P", _three: "3q", _two: "2q"}
    packer = struct.Struct("@" + "".join(codes[kind] for _, kind in structure._fields_) + "0q")
    assert packer.size == ctypes.sizeof(structure)
    return packer


PACK_RULE, PACK_GRADIENTS, PACK_NORM = (_packer(s).pack for s in (DeltaRule, DeltaGradients, QkNorm))

_lib.navi_policy_last_error.restype = ctypes.c_char_p
_lib.navi_policy_last_error.argtypes = []
# (structures as bytes or by reference)
for _name in ("navi_delta_forward", "navi_delta_step", "navi_qk_norm", "navi_qk_norm_backward"):
    getattr(_lib, _name).restype = ctypes.c_int
    getattr(_lib, _name).argtypes = [_vp, _vp]
for _name in ("navi_delta_scratch", "navi_delta_workspace", "navi_qk_norm_workspace"):
    getattr(_lib, _name).restype = _i64
    getattr(_lib, _name).argtypes = [_vp]
_lib.navi_delta_backward.restype = ctypes.c_int
_lib.navi_delta_backward.argtypes = [_vp, _vp, _vp]
_lib.navi_clip_grad_norm.restype = ctypes.c_int
_lib.navi_clip_grad_norm.argtypes = [_i32, _vp, _vp, _vp, _vp, _f32, _f32, _vp, _vp, _vp]


def lib() -> ctypes.CDLL:
    return _lib


def last_error() -> str:
    return _lib.navi_policy_last_error().decode(errors="replace")


def check(code: int) -> int:
    """Raise ``RuntimeError`` for a failed call; a size (a code >= 0) is returned."""
    if code < 0:
        raise RuntimeError(last_error() or f"navi_policy call failed with code {code}")
    return code

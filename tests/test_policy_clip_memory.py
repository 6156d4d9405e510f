"""``navi_clip_grad_norm`` refuses tensors that share memory before any launch (a workgroup would
read what another has scaled): addresses that are never read, no GPU."""

from __future__ import annotations

import ctypes

import pytest

native = pytest.importorskip("navi_amd._policy_native")


def clip(tensors):
    """The entry point's code and message for (from, to, count, dtype) of each tensor."""
    n = len(tensors)
    of = lambda kind, i: (kind * n)(*[t[i] for t in tensors])  # noqa: E731
    code = native.lib().navi_clip_grad_norm(n, of(ctypes.c_void_p, 0), of(ctypes.c_void_p, 1), of(ctypes.c_int64, 2),
                                            of(ctypes.c_int32, 3), 1.0, 1e-6, 4096, 4096, None)
    return code, native.last_error()


F32, BF16 = native.F32, native.BF16
A, B, C = 1 << 20, 2 << 20, 3 << 20


@pytest.mark.parametrize("tensors, words", [
    ([(A, A, 10, F32), (A, A, 10, F32)], "tensors 0 and 1 that are written"),  # named twice, in place
    ([(C, C, 10, F32), (B, B, 4, BF16), (C, C, 10, F32)], "tensors 0 and 2 that are written"),
    ([(A, A, 10, F32), (A + 36, A + 36, 10, F32)], "tensors 0 and 1 that are written"),  # the last number
    ([(A + 18, A + 18, 10, BF16), (A, A, 10, BF16)], "tensors 0 and 1 that are written"),
    ([(A, C, 10, F32), (B, C, 10, F32)], "tensors 0 and 1 that are written"),  # one output for two
    ([(A, A + 4, 10, F32)], "tensor 0 that is read and tensor 0 that is written"),  # moved by one number
    ([(A + 4, A, 10, F32)], "tensor 0 that is read and tensor 0 that is written"),
    ([(A, B, 10, F32), (B, C, 10, F32)], "tensor 1 that is read and tensor 0 that is written"),
    ([(A, C, 10, F32), (B, A + 36, 1, F32)], "tensor 0 that is read and tensor 1 that is written"),
    ([(A, B, 1, F32), (C, C, 2000000, F32), (C + 7999996, 16 << 20, 1, F32)], "tensor 2 that is read and tensor 1 that is written"),
    ([(A, A, 10, F32)] + [(B + 64 * i, B + 64 * i, 16, F32) for i in range(300)] + [(A, A, 1, F32)],
     "tensors 0 and 301 that are written"),
])
def test_shared_memory_is_refused(tensors, words):
    code, message = clip(tensors)
    assert code == native.NAVI_POLICY_E_ARG and words in message

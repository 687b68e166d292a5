"""Refusals of the attention entry points of the C-ABI that need no GPU: every call
here has to end before a launch."""

import ctypes
from pathlib import Path

import pytest
import torch  # noqa: F401  (binds the HIP runtime torch ships before the library loads)

LIB = Path(__file__).resolve().parents[1] / "torchlib-xpu_amd" / "mx_fbgemm" / "lib" / "libmx_fbgemm_kernels.so"
EINVAL = -1


class Tensor3(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("row_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64)]


class Problem(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int32), ("index_bytes", ctypes.c_int32), ("q_offsets", ctypes.c_void_p),
                ("k_offsets", ctypes.c_void_p), ("B", ctypes.c_int64), ("Nq", ctypes.c_int64),
                ("Nk", ctypes.c_int64), ("H", ctypes.c_int32), ("Hkv", ctypes.c_int32), ("D", ctypes.c_int32),
                ("causal", ctypes.c_int32), ("scale", ctypes.c_float)]


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(str(LIB))
    P, T3, Z = ctypes.c_void_p, ctypes.POINTER(Tensor3), ctypes.c_size_t
    lib.mx_last_error.restype = ctypes.c_char_p
    lib.mx_jagged_attention_forward.argtypes = [ctypes.POINTER(Problem), T3, T3, T3, P, P, P, Z, P]
    lib.mx_jagged_attention_backward.argtypes = [ctypes.POINTER(Problem), T3, T3, T3, T3, T3, P, P, P, P, P, Z, P]
    return lib


# Never read: a call that took it for an address on the device would not return EINVAL.
BUFFER = ctypes.create_string_buffer(1 << 16)
HERE = (ctypes.addressof(BUFFER) + 63) // 64 * 64


def both(lib, p):
    """Status of the forward and of the backward."""
    t = Tensor3(HERE, p.H * p.D, p.D)
    f = lib.mx_jagged_attention_forward(p, t, t, t, HERE, HERE, HERE, 1 << 15, None)
    b = lib.mx_jagged_attention_backward(p, t, t, t, t, t, HERE, HERE, HERE, HERE, HERE, 1 << 15, None)
    return f, b


@pytest.mark.parametrize("B,Nq,Nk", [(0, 5, 5), (0, 5, 0), (0, 0, 5), (3, 0, 0), (3, 5, 5)])
@pytest.mark.parametrize("which", ["both", "q_offsets", "k_offsets"])
def test_rows_or_lists_without_offsets_are_refused(lib, B, Nq, Nk, which):
    """Without lists the offsets still have one entry, which the kernels read."""
    p = Problem(2, 8, HERE, HERE, B, Nq, Nk, 2, 2, 32, 1, 0.25)
    for name in ("q_offsets", "k_offsets") if which == "both" else (which,):
        setattr(p, name, None)
    assert both(lib, p) == (EINVAL, EINVAL)
    assert b"offsets" in lib.mx_last_error()


def test_nothing_at_all_needs_no_offsets(lib):
    f, b = both(lib, Problem(2, 8, None, None, 0, 0, 0, 2, 2, 32, 1, 0.25))
    assert f == 0 and b != EINVAL  # (the backward asks the device for its state, which may not be there)

"""Refusals of the C-ABI's rotation, row and 4-bit cache entry points that need no
GPU (every call here has to end before a launch), and the plain forms themselves."""

import ctypes
from pathlib import Path

import numpy as np
import pytest
import torch

import oracle as orc
from mx_fbgemm.sequence_attention import PagedSequenceCache, rotary_table
from rows_helpers import angles, attention4, make, page_table, rotate, rows4, values4

LIB = Path(__file__).resolve().parents[1] / "torchlib-xpu_amd" / "mx_fbgemm" / "lib" / "libmx_fbgemm_kernels.so"
EINVAL, F32, F16, BF16 = -1, 0, 1, 2
P, I32, I64, F, Z = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float, ctypes.c_size_t


class Tensor3(ctypes.Structure):
    _fields_ = [("data", P), ("row_stride", I64), ("head_stride", I64)]


class Cache(ctypes.Structure):
    _fields_ = [("k", P), ("v", P), *[(n, I64) for n in ("kp", "ks", "kh", "vp", "vs", "vh")], ("pages", I64),
                ("page_size", I32), ("table", P), ("table_row_stride", I64), ("table_width", I64)]


class Rotary(ctypes.Structure):
    _fields_ = [("table", P), ("positions", I64), ("pairs", I32), ("interleaved", I32)]


# Never read: a call that took it for an address on the device would not return EINVAL.
BUFFER = ctypes.create_string_buffer(1 << 12)
HERE = (ctypes.addressof(BUFFER) + 63) // 64 * 64


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(str(LIB))
    T, C, R = ctypes.POINTER(Tensor3), ctypes.POINTER(Cache), ctypes.POINTER(Rotary)
    lib.mx_last_error.restype = ctypes.c_char_p
    lib.mx_jagged_rotary.argtypes = [I32, T, I64, I32, I32, R, I32, I64, P, I32, P, I32, P, P]
    lib.mx_paged_cache_append_rows.argtypes = [C, I32, I32, I32, I32, I32, T, T, T, R, I64, I64, P, I32, P, I32, P, P]
    lib.mx_paged_cache_gather.argtypes = [C, I32, I32, I32, I32, I64, I64, P, I32, P, P, P]
    lib.mx_paged_cache_attention_int4.argtypes = [C, I32, T, I64, I32, I32, I32, P, I32, F, P, P, Z, P]
    lib.mx_paged_cache_attention_int4_workspace_bytes.argtypes = [C, I64, I32, I32, I32]
    lib.mx_paged_cache_attention_int4_workspace_bytes.restype = Z
    return lib


def rows():
    return Tensor3(HERE, 64, 32)


def cache(**kw):
    c = Cache(HERE, HERE, 640, 40, 20, 640, 40, 20, 2, 16, HERE, 3, 3)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def rotary(**kw):
    return Rotary(**{**dict(table=HERE, positions=10, pairs=16, interleaved=0), **kw})


def test_rotary(lib):
    base = [BF16, rows(), 4, 2, 32, rotary(), 0, 2, HERE, 8, HERE, 8, HERE, None]
    for at, bad in [(0, F32), (1, None), (1, Tensor3(HERE + 8, 64, 32)), (1, Tensor3(HERE, 60, 32)),
                    (1, Tensor3(None, 64, 32)), (1, Tensor3(HERE, 64, -32)), (2, -1), (3, -1), (3, 1 << 20), (4, 36),
                    (4, 136), (4, 0), (5, None), (5, rotary(pairs=0)), (5, rotary(pairs=6)), (5, rotary(pairs=20)),
                    (5, rotary(positions=-1)), (5, rotary(positions=1 << 31)), (5, rotary(table=None)),
                    (5, rotary(table=HERE + 4)), (7, -1), (8, None), (9, 2), (11, 2), (12, None), (12, HERE + 8)]:
        args = list(base)
        args[at] = bad
        assert lib.mx_jagged_rotary(*args) == EINVAL, (at, bad)
        assert lib.mx_last_error()
    args = list(base)
    args[2] = 0
    assert lib.mx_jagged_rotary(*args) == 0  # nothing to do


def test_append_rows(lib):
    base = [cache(), 4, F16, 2, 2, 32, rows(), rows(), rows(), rotary(), 4, 2, HERE, 8, HERE, 8, HERE, None]
    for at, bad in [(0, None), (0, cache(page_size=0)), (0, cache(pages=-1)), (0, cache(k=None)), (0, cache(v=HERE + 2)),
                    (0, cache(kh=18)), (0, cache(vp=-4)), (0, cache(table=None)), (0, cache(table_width=-1)), (1, 8),
                    (1, 0), (2, F32), (3, -1), (3, 1 << 20), (4, 0), (5, 12), (6, None), (7, None), (8, None),
                    (8, Tensor3(HERE + 4, 64, 32)), (9, None), (9, rotary(pairs=20)), (10, -1), (11, -1), (12, None),
                    (13, 3), (14, None), (15, 5), (16, None)]:
        args = list(base)
        args[at] = bad
        assert lib.mx_paged_cache_append_rows(*args) == EINVAL, (at, bad)
    args = list(base)  # 16 bits want 16 bytes: strides of 4 elements are no multiple of 8
    args[1] = 16
    assert lib.mx_paged_cache_append_rows(*args) == EINVAL
    args = list(base)
    args[10] = 0
    assert lib.mx_paged_cache_append_rows(*args) == 0


def test_gather(lib):
    base = [cache(), 4, F16, 2, 32, 4, 2, HERE, 8, HERE, HERE, None]
    for at, bad in [(0, None), (0, cache(ks=2)), (0, cache(table=None)), (1, 2), (2, F32), (3, 0), (4, 20), (5, -1), (6, -1),
                    (7, None), (8, 1), (9, None), (10, None), (10, HERE + 8)]:
        args = list(base)
        args[at] = bad
        assert lib.mx_paged_cache_gather(*args) == EINVAL, (at, bad)
    args = list(base)
    args[5] = 0
    assert lib.mx_paged_cache_gather(*args) == 0


def test_attention(lib):
    base = [cache(), BF16, rows(), 3, 4, 2, 32, HERE, 8, 0.5, HERE, None, 0, None]
    for at, bad in [(0, None), (0, cache(kh=6)), (0, cache(page_size=-1)), (0, cache(table_width=1 << 30)), (1, F32),
                    (2, None), (2, Tensor3(HERE, 60, 32)), (3, -1), (3, 1 << 31), (4, 3), (4, 0), (5, 0), (6, 12), (6, 136),
                    (7, None), (8, 2), (9, 0.0), (9, float("inf")), (9, float("nan")), (10, None)]:
        args = list(base)
        args[at] = bad
        assert lib.mx_paged_cache_attention_int4(*args) == EINVAL, (at, bad)
    args = list(base)
    args[3] = 0
    assert lib.mx_paged_cache_attention_int4(*args) == 0
    for bad in ((None, 3, 4, 2, 32), (cache(), 0, 4, 2, 32), (cache(), 3, 3, 2, 32), (cache(), 3, 4, 0, 32)):
        assert lib.mx_paged_cache_attention_int4_workspace_bytes(*bad) == 0


# -- the plain forms -----------------------------------------------------------

def test_table_and_rotation():
    t = rotary_table(50, 16, device="cpu")
    assert t.shape == (50, 8, 2) and t.dtype == torch.float32 and torch.equal(t, angles(50, 16))
    for bad in ((-1, 16), (5, 12), (5, 0)):
        with pytest.raises(ValueError):
            rotary_table(*bad, device="cpu")
    with pytest.raises(ValueError):
        rotary_table(5, 16, base=0.0, device="cpu")
    x = make((50, 2, 24), torch.float64, 1)
    for inter in (False, True):
        y = rotate(x, [0, 50], t.double(), None, inter, dtype=torch.float64)
        back = rotate(y, [0, 50], t.double(), None, inter, -1, torch.float64)
        assert torch.allclose(back, x, atol=1e-6) and torch.equal(y[..., 16:], x[..., 16:])
        # Scores depend on the distance of the positions alone.
        k = rotate(x[:1].expand(50, 2, 24), [0, 50], t.double(), None, inter, dtype=torch.float64)
        s = (k[5:, 0] * k[:-5, 0]).sum(-1)
        assert torch.allclose(s, s[:1].expand_as(s), atol=1e-5)


def test_rows_of_four_bits():
    x = make((7, 3, 40), torch.float32, 1)
    r = rows4(x)
    assert r.shape == (7, 3, 24)
    v = values4(r)
    want = orc.dequantize_fused_nbit(r.reshape(21, 24).numpy(), 4, 40).reshape(7, 3, 40)
    assert np.array_equal(v.astype(np.float32), want)
    spread = (x.amax(-1) - x.amin(-1)).numpy()[..., None]
    # Half a step; scale's and bias's fp16 roundings, at most fifteen times over.
    assert (np.abs(v - x.numpy()) <= spread / 30 + 16 * 2.0 ** -11 * np.abs(x.numpy()).max()).all()


def test_attention_of_four_bits_is_that_of_its_values():
    q = make((2, 4, 16), torch.float64, 1).numpy()
    ks, vs = ([rows4(make((n, 2, 16), torch.float32, s + n)) for n in (5, 9)] for s in (1, 2))
    out, tol = attention4(q, ks, vs, 0.25, "float16")
    for b in range(2):
        for h in range(4):
            k, v = values4(ks[b])[:, h // 2], values4(vs[b])[:, h // 2]
            p = torch.softmax(torch.from_numpy(k @ q[b, h] * 0.25), 0).numpy()
            assert np.allclose(out[b, h], p @ v, atol=1e-12)
    assert (tol > 0).all() and (tol < 2e-2).all()


def test_page_tables():
    t, pages = page_table([5, 0, 9], 4, extra=2)
    assert t.shape == (3, 3) and pages == 7
    used = t[t >= 0].tolist()
    assert len(set(used)) == len(used) == 5 and (t[1] == -1).all()


# -- the cache object's host side -------------------------------------------------

def make_cache(**kw):
    args = dict(pages=6, page_size=4, heads=2, head_dim=16, max_sequences=3, max_length=16, device="cpu")
    return PagedSequenceCache(**{**args, **kw})


def test_cache_of_four_bits():
    c = make_cache(bits=4)
    assert c.k.dtype == torch.uint8 and c.k.shape == (6, 4, 2, 12) and c.k.stride() == (96, 12, 48, 1)
    assert c.bits == 4 and c.dtype == torch.bfloat16
    a = c.add()
    with pytest.raises(ValueError, match="rows are"):
        c.append([a], [1], torch.zeros((1, 2, 16)), torch.zeros((1, 2, 16)))
    for bits in (8, 0, 2):
        with pytest.raises(ValueError):
            make_cache(bits=bits)


def test_cache_with_positions():
    t = rotary_table(16, 16, device="cpu")
    c = make_cache(rotary=t)
    k = torch.zeros((2, 2, 16), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="q has 1 rows"):
        c.append([c.add()], [2], k, k, k[:1])
    assert make_cache().append([], [], k[:0], k[:0], k[:0]).shape == (0, 2, 16)
    for bad in (t[:15], t.double(), t[:, :3], t[:, :, :1], t[0], angles(16, 24), t[:, :0]):
        with pytest.raises(ValueError):
            make_cache(rotary=bad)

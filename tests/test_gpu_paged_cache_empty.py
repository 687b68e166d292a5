"""Sequences without tokens beside others, in every way that a call's sequences are
cut over blocks: their outputs are zeros, the others' are their own, and nothing
outside the arguments is read into a result or written.

lengths, the table and q are slices of longer tensors: what follows them looks like
more sequences with tokens."""

import ctypes
from pathlib import Path

import numpy as np
import pytest
import torch

from attention_helpers import check, paged_attention
from test_gpu_paged_cache import make, make_cache

pytestmark = pytest.mark.gpu

LIB = Path(__file__).resolve().parents[1] / "torchlib-xpu_amd" / "mx_fbgemm" / "lib" / "libmx_fbgemm_kernels.so"
OPS = torch.ops.mx_fbgemm
PAGE = 16

# Sequences of no, one and two tiles of a block (0, 1, 2): empty ones first, in the
# middle, last, several in a row, and nothing else.
MIXES = [(0, 2, 1), (0, 1, 2), (1, 0, 2), (2, 0, 0, 1), (2, 1, 0), (1, 2, 0, 0), (0, 2, 0), (0, 0, 0), (0,)]


class Tensor3(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("row_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64)]


class Cache(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p),
                ("k_page", ctypes.c_int64), ("k_slot", ctypes.c_int64), ("k_head", ctypes.c_int64),
                ("v_page", ctypes.c_int64), ("v_slot", ctypes.c_int64), ("v_head", ctypes.c_int64),
                ("pages", ctypes.c_int64), ("page_size", ctypes.c_int32), ("table", ctypes.c_void_p),
                ("table_row", ctypes.c_int64), ("width", ctypes.c_int64)]


def plan_of(name, mix):
    """Lengths, heads (query, key-value), width and the table's room that have a call cut
    this way: a block of four waves per sequence and head where there are 2048 of
    them, or where no table holds more than one tile; a block of 16 or 8 waves where
    it holds at most two of their tiles; else shares."""
    tile = {"plain": 128, "one_tile": 128, "wide": 512, "wide_128": 256, "shares": 128}[name]
    D = 128 if name == "wide_128" else 64 if name == "wide" else 32
    room = {"plain": 4, "one_tile": 1, "wide": 2, "wide_128": 2, "shares": 12}[name] * tile
    size = {0: 0, 1: tile - 3, 2: tile + 48 if name != "one_tile" else tile}  # whole pages
    lengths = [size[m] for m in mix]
    H, Hkv = (4, 2) if name != "plain" else (64, 64)
    if name == "plain":
        lengths = lengths * -(-32 // len(lengths))  # 64 heads of 32 sequences: 2048 blocks
    return lengths, H, Hkv, D, room


def call(dev, lengths, H, Hkv, D, room, index):
    """The sequences' arguments as slices, and what they have to give."""
    kc, vc, table, ks, vs = make_cache(lengths, PAGE, Hkv, D, "bfloat16")
    B = len(lengths)
    q = make((B, H, D), "bfloat16", 99)
    # More sequences behind the last: full ones, on pages of the cache.
    wide = torch.zeros((B + 4, room // PAGE), dtype=torch.int32)
    wide[:B] = -1
    wide[:B, : table.size(1)] = table
    more = torch.full((B + 4,), room, dtype=index)
    more[:B] = torch.tensor(lengths, dtype=index)
    qs = torch.cat([q, make((4, H, D), "bfloat16", 98)])
    want, tol = paged_attention(q.double().numpy(), [k.double().numpy() for k in ks],
                                [v.double().numpy() for v in vs], D ** -0.5, "bfloat16")
    return (qs.to(dev)[:B], kc.to(dev), vc.to(dev), wide.to(dev)[:B], more.to(dev)[:B]), want, tol


@pytest.mark.parametrize("mix", MIXES, ids=lambda m: "".join(map(str, m)))
@pytest.mark.parametrize("plan", ["plain", "one_tile", "wide", "wide_128", "shares"])
def test_empty_sequences(dev, plan, mix):
    lengths, H, Hkv, D, room = plan_of(plan, mix)
    index = torch.int32 if len(mix) % 2 else torch.int64
    print(f"[case] {plan} lengths={lengths[:4]} of {len(lengths)} room={room}", flush=True)
    args, want, tol = call(dev, lengths, H, Hkv, D, room, index)
    out = OPS.paged_cache_attention(*args)
    check(out.double().cpu().numpy(), want, tol, "out")
    for b, n in enumerate(lengths):
        if n == 0:
            assert torch.count_nonzero(out[b]) == 0
    assert torch.equal(OPS.paged_cache_attention(*args), out)


@pytest.mark.parametrize("mix", [(0, 2, 1), (2, 0, 1), (2, 1, 0), (0, 0)], ids=lambda m: "".join(map(str, m)))
@pytest.mark.parametrize("plan", ["plain", "one_tile", "wide", "wide_128", "shares"])
def test_nothing_outside_is_written(dev, plan, mix):
    """The C entry with an output and a workspace between guards; the plans that need no
    workspace get none."""
    lib = ctypes.CDLL(str(LIB))
    P, i32, i64, size = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_size_t
    lib.mx_last_error.restype = ctypes.c_char_p
    lib.mx_paged_cache_attention_workspace_bytes.restype = size
    lib.mx_paged_cache_attention_workspace_bytes.argtypes = [ctypes.POINTER(Cache), i64, i32, i32, i32]
    lib.mx_paged_cache_attention.argtypes = [ctypes.POINTER(Cache), i32, ctypes.POINTER(Tensor3), i64, i32, i32,
                                             i32, P, i32, ctypes.c_float, P, P, size, P]
    lengths, H, Hkv, D, room = plan_of(plan, mix)
    B = len(lengths)
    print(f"[case] {plan} lengths={lengths[:4]} of {B} through ctypes", flush=True)
    (q, kc, vc, table, n), want, tol = call(dev, lengths, H, Hkv, D, room, torch.int64)
    c = Cache(kc.data_ptr(), vc.data_ptr(), kc.stride(0), kc.stride(1), kc.stride(2), vc.stride(0), vc.stride(1),
              vc.stride(2), kc.size(0), PAGE, table.data_ptr(), table.stride(0), table.size(1))
    need = lib.mx_paged_cache_attention_workspace_bytes(c, B, H, Hkv, D)
    assert (need > 0) == (plan == "shares")
    guard = 4096
    room_out = torch.full((guard + B * H * D + guard,), 7.0, dtype=torch.bfloat16, device=dev)
    out = room_out[guard: guard + B * H * D].view(B, H, D)
    ws = torch.full((guard + need + guard,), 7, dtype=torch.uint8, device=dev)
    q3 = Tensor3(q.data_ptr(), q.stride(0), q.stride(1))
    rc = lib.mx_paged_cache_attention(c, 2, q3, B, H, Hkv, D, n.data_ptr(), 8, D ** -0.5, out.data_ptr(),
                                      ws.data_ptr() + guard if need else None, need,
                                      torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.mx_last_error()
    check(out.double().cpu().numpy(), want, tol, "out")
    for x, edge in ((room_out, 7.0), (ws, 7)):
        assert bool((x[:guard] == edge).all()) and bool((x[x.numel() - guard:] == edge).all())


def test_lengths_below_zero_and_past_the_table(dev):
    """A length below zero is none, one past the table's room is the room, in each plan."""
    for plan in ("plain", "one_tile", "wide", "wide_128", "shares"):
        lengths, H, Hkv, D, room = plan_of(plan, (0, 2, 0))
        print(f"[case] {plan}", flush=True)
        args, want, tol = call(dev, lengths, H, Hkv, D, room, torch.int64)
        n = args[4]
        n[0], n[len(lengths) - 1] = -2 ** 62, -1
        check(OPS.paged_cache_attention(*args).double().cpu().numpy(), want, tol, plan)
        n[1] = 2 ** 62  # the table's entries behind its own are -1: absent
        check(OPS.paged_cache_attention(*args).double().cpu().numpy(), want, tol, plan)

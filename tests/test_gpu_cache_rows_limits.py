"""Rows whose positions pass 64 bits, and rows that hold no number: what appends,
rotation and reading back make of them, on the GPU."""

import pytest
import torch

from rows_helpers import angles, make

pytestmark = pytest.mark.gpu

OPS = torch.ops.mx_fbgemm
FAR = [2 ** 63 - 1, 2 ** 63 - 2, 2 ** 63 - 5, 2 ** 62]


@pytest.mark.parametrize("H", [1, 20])
@pytest.mark.parametrize("start", FAR)
def test_rotation_at_positions_past_64_bits(dev, H, start):
    """Lists of several rows: start + i wraps around in 64 bits; none has an angle."""
    x = make((14, H, 32), "bfloat16", 1).to(dev)
    off = torch.tensor([0, 9, 14], device=dev)
    t = angles(20, 32).to(dev)
    y = OPS.jagged_rotary(x, off, t, torch.tensor([start, 3], device=dev))
    assert torch.isnan(y[:9]).all()
    assert torch.equal(y[9:], OPS.jagged_rotary(x[9:].contiguous(), torch.tensor([0, 5], device=dev), t,
                                                   torch.tensor([3], device=dev)))


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("rotary", [False, True])
@pytest.mark.parametrize("start", FAR)
def test_appends_at_positions_past_64_bits(dev, four, rotary, start):
    """Their rows are dropped; those of the lists around them are not."""
    page, Hkv, D = 4, 2, 32
    k = make((12, Hkv, D), "float16", 1).to(dev)
    off = torch.tensor([0, 2, 9, 12], device=dev)
    table = torch.tensor([[0, 1], [2, 3], [4, 5]], dtype=torch.int32, device=dev)
    t = angles(8, D).to(dev)

    def append(starts, rows, offsets, tab):
        kc, vc = (torch.zeros((6, page, Hkv, D // 2 + 4 if four else D), device=dev,
                              dtype=torch.uint8 if four else torch.float16) for _ in range(2))
        args = (rows, rows, offsets, torch.tensor(starts, device=dev))
        if rotary:
            OPS.paged_cache_append_rotary(None, *args, t, kc, vc, tab)
        else:
            OPS.paged_cache_append(*args, kc, vc, tab)
        return kc, vc

    got = append([1, start, 3], k, off, table)
    keep = torch.cat([k[:2], k[9:]])
    want = append([1, 3], keep, torch.tensor([0, 2, 5], device=dev), table[[0, 2]])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.count_nonzero(got[0][2:4]) == 0 and torch.count_nonzero(got[0][:2]) > 0


@pytest.mark.parametrize("first", [-2 ** 63, -2 ** 63 + 3, -2 ** 62])
def test_offsets_below_every_row(dev, first):
    """The rows lie further behind the first offset than 63 bits tell."""
    x = make((6, 2, 32), "float16", 1).to(dev)
    off, zero = torch.tensor([first, 6], device=dev), torch.zeros(1, dtype=torch.int64, device=dev)
    t = angles(20, 32).to(dev)
    assert torch.isnan(OPS.jagged_rotary(x, off, t, zero)).all()
    assert torch.isnan(OPS.jagged_rotary(x, off, t)).all()
    kc = torch.zeros((2, 4, 2, 20), dtype=torch.uint8, device=dev)
    table = torch.zeros((1, 2), dtype=torch.int32, device=dev)
    OPS.paged_cache_append(x, x, off, zero, kc, kc.clone(), table)
    assert torch.count_nonzero(kc) == 0
    kc[..., -4:] = 1
    k, v = OPS.paged_cache_gather(kc, kc, table, off, 6, torch.float16)
    assert torch.count_nonzero(k) == 0 and torch.count_nonzero(v) == 0

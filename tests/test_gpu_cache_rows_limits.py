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


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [8, 40, 64, 96, 128])
@pytest.mark.parametrize("rotary", [False, True])
def test_nan_of_an_element_is_its_heads_row(dev, dtype, D, rotary):
    """A 4-bit row has no code for NaN: the head's whole row is NaN (scale and bias,
    codes 0), where a 16-bit cache shows the element.  Other heads' and tokens' rows
    are those of the same values without it."""
    n, Hkv = D + 2, 3
    k, v = (make((n, Hkv, D), dtype, s).to(dev) for s in (1, 2))
    bad_k, bad_v = k.clone(), v.clone()
    for i in range(D):
        bad_k[i, 1, i] = float("nan")
        bad_v[i, 2, D - 1 - i] = float("nan")
    bad_k[D, 0] = float("nan")
    page = 16
    pages = -(-n // page)
    table = torch.arange(pages, dtype=torch.int32, device=dev).view(1, pages)
    off, zero, t = torch.tensor([0, n], device=dev), torch.tensor([0], device=dev), angles(n, D).to(dev)

    def append(k, v):
        kc, vc = (torch.zeros((pages, page, Hkv, D // 2 + 4), dtype=torch.uint8, device=dev) for _ in range(2))
        if rotary:
            OPS.paged_cache_append_rotary(None, k, v, off, zero, t, kc, vc, table)
        else:
            OPS.paged_cache_append(k, v, off, zero, kc, vc, table)
        return kc, vc

    got, want = append(bad_k, bad_v), append(k, v)
    read = OPS.paged_cache_gather(*got, table, off, n, torch.bfloat16)
    for c, w, x, r in zip(got, want, (bad_k, bad_v), read):
        bad = torch.isnan(x).any(-1)
        c, w = (y.view(-1, Hkv, D // 2 + 4)[:n] for y in (c, w))
        assert torch.equal(c[~bad], w[~bad])
        assert torch.count_nonzero(c[bad][:, :-4]) == 0
        assert torch.isnan(c[bad][:, -4:].contiguous().view(torch.float16)).all()
        assert torch.equal(torch.isnan(r), bad[..., None].expand_as(r))
    # And attention shows it, in the heads that read it.
    q = make((1, 2 * Hkv, D), dtype, 3).to(dev)
    out = OPS.paged_cache_attention(q, *got, table, torch.tensor([n - 1], device=dev))
    assert torch.isnan(out).all()
    out = OPS.paged_cache_attention(q, got[0], want[1], table, torch.tensor([D], device=dev))
    assert torch.isnan(out[0]).all(-1).tolist() == [False, False, True, True, False, False]
    assert torch.isnan(out[0]).any(-1).tolist() == [False, False, True, True, False, False]


@pytest.mark.parametrize("dtype,value", [(torch.float16, float("inf")), (torch.float16, -float("inf")),
                                         (torch.bfloat16, float("inf")), (torch.bfloat16, -float("inf")),
                                         (torch.bfloat16, -70000.0), (torch.bfloat16, 1.5e6), (torch.bfloat16, 3e38)])
def test_what_fp16_does_not_hold_reads_back_as_nan(dev, dtype, value):
    """Infinities, a smallest value below fp16's range, and a range whose fifteenth is past it."""
    D = 32
    x = make((2, 1, D), dtype, 1).to(dev)
    x[0, 0, 5] = value
    kc = torch.zeros((1, 2, 1, D // 2 + 4), dtype=torch.uint8, device=dev)
    vc, table, off = kc.clone(), torch.zeros((1, 1), dtype=torch.int32, device=dev), torch.tensor([0, 2], device=dev)
    OPS.paged_cache_append(x, x, off, off[:1], kc, vc, table)
    k, v = OPS.paged_cache_gather(kc, vc, table, off, 2, torch.bfloat16)
    assert torch.isnan(k[0]).all() and torch.isnan(v[0]).all() and torch.isfinite(k[1]).all()
    q = make((1, 1, D), dtype, 2).to(dev)
    assert torch.isnan(OPS.paged_cache_attention(q, kc, vc, table, torch.tensor([2], device=dev))).all()


def test_values_past_fp16_whose_range_it_holds(dev):
    x = make((1, 1, 32), torch.bfloat16, 1).to(dev)
    x[0, 0, 5] = 90112.0  # a scale of 6,000: 15 steps reach it
    kc = torch.zeros((1, 1, 1, 20), dtype=torch.uint8, device=dev)
    table, off = torch.zeros((1, 1), dtype=torch.int32, device=dev), torch.tensor([0, 1], device=dev)
    OPS.paged_cache_append(x, x, off, off[:1], kc, kc.clone(), table)
    k, _ = OPS.paged_cache_gather(kc, kc, table, off, 1, torch.bfloat16)
    # Scale and bias are rounded to fp16 (2^-11), the value to bf16 (2^-8).
    assert abs(float(k[0, 0, 5]) - 90112.0) <= 90112.0 * (2 ** -10 + 2 ** -8) and torch.isfinite(k).all()

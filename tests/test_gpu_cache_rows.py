"""Appends that rotate, caches of 4-bit rows and lists read back, on the GPU: bit for
bit against plain forms, and their refusals."""

import numpy as np
import pytest
import torch

from rows_helpers import DT, angles, make, page_table, rotate, rows4, values4

pytestmark = pytest.mark.gpu

OPS = torch.ops.mx_fbgemm


def bits(x):
    x = x.detach().cpu().contiguous()
    return x if x.dtype == torch.uint8 else x.view(torch.int16)


def empty_cache(pages, page, Hkv, D, dtype, four, seed=0, head_major=False):
    """A cache full of noise; 4-bit rows of any bytes."""
    if not four:
        return make((pages, page, Hkv, D), dtype, seed)
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, 256, (pages, page, Hkv, D // 2 + 4), generator=g, dtype=torch.uint8)


def put(cache, rows, table, offsets, starts, page, four):
    """rows (fp32 [N, Hkv, D]) into a copy of the cache, token by token."""
    c = cache.clone()
    r = rows4(rows) if four else rows.to(c.dtype)
    for b in range(len(offsets) - 1):
        for i in range(offsets[b], offsets[b + 1]):
            t = starts[b] + i - offsets[b]
            if 0 <= t // page < table.shape[1] and starts[b] >= 0:
                p = int(table[b, t // page])
                if 0 <= p < c.shape[0] and not torch.isnan(rows[i]).any():
                    c[p, t % page] = r[i]
    return c


def run(dev, n, starts, page, H, Hkv, D, dtype, four, R=None, interleaved=False, index=torch.int64, place=lambda c: c,
        extra_rows=0, positions=None):
    """One append; R None: without rotation."""
    print(f"[case] {len(n)} lists of {sum(n)} rows page={page} H={H}/{Hkv} D={D} R={R} {dtype} four={four}", flush=True)
    off = np.concatenate([[0], np.cumsum(n)]).astype(int).tolist()
    table, pages = page_table([a + b for a, b in zip(n, starts)], page, seed=len(n))
    N = off[-1] + extra_rows
    q, k, v = (make((N, h, D), dtype, s) for h, s in ((H, 1), (Hkv, 2), (Hkv, 3)))
    kc, vc = (empty_cache(pages, page, Hkv, D, dtype, four, s) for s in (4, 5))
    kd, vd = place(kc.to(dev)), place(vc.to(dev))
    o, s = (torch.tensor(x, dtype=index, device=dev) for x in (off, starts))
    td = table.to(dev)
    if R is None:
        OPS.paged_cache_append(k.to(dev), v.to(dev), o, s, kd, vd, td)
        kr = k.float()
    else:
        most = positions if positions is not None else max(a + b for a, b in zip(n, starts)) + 1
        t = angles(most, R)
        qr = OPS.paged_cache_append_rotary(q.to(dev) if H else None, k.to(dev), v.to(dev), o, s, t.to(dev), kd, vd, td,
                                           interleaved)
        assert qr.shape == (N, H, D)
        want = rotate(q, off, t, starts, interleaved).to(DT[dtype])
        nan = torch.isnan(want)
        assert torch.equal(torch.isnan(qr.cpu()), nan)
        assert torch.equal(bits(qr.cpu().masked_fill(nan, 0)), bits(want.masked_fill(nan, 0)))
        kr = rotate(k, off, t, starts, interleaved)
    vr = v.float()
    if R is not None and positions is not None:
        vr = torch.where(torch.isnan(kr).any(-1, keepdim=True), float("nan"), vr)
    assert torch.equal(bits(kd), bits(put(kc, kr, table, off, starts, page, four)))
    assert torch.equal(bits(vd), bits(put(vc, vr, table, off, starts, page, four)))
    return kd, vd, td, table


def heads_first(c):
    return c.transpose(1, 2).contiguous().transpose(1, 2)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("D,R", [(8, 8), (16, 8), (24, 24), (40, 40), (64, 64), (64, 24), (72, 72), (96, 96), (104, 48),
                                 (128, 128), (128, 64)])
def test_widths(dev, dtype, four, D, R):
    run(dev, [3, 0, 30, 1], [5, 2, 0, 9], 16, 4, 2, D, dtype, four, R, interleaved=D in (24, 64, 128))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("D", [8, 32, 40, 64, 88, 96, 128])
def test_four_bits_without_rotation(dev, dtype, D):
    run(dev, [3, 0, 30, 1], [5, 2, 0, 9], 16, 0, 2, D, dtype, True)


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("H,Hkv", [(0, 1), (1, 1), (8, 1), (32, 8), (3, 5), (130, 2)])
def test_heads(dev, four, H, Hkv):
    run(dev, [2, 5, 1], [0, 7, 100], 16, H, Hkv, 64, "bfloat16", four, 64)


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("page", [1, 3, 5, 16, 100])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_pages(dev, four, page, index):
    rng = np.random.default_rng(page)
    n, starts = ([int(v) for v in rng.integers(0, m, 90)] for m in (7, 40))
    run(dev, n, starts, page, 2, 2, 32, "float16", four, 32, index=index)


@pytest.mark.parametrize("four", [False, True])
def test_many_lists_and_long_ones(dev, four):
    run(dev, [1] * 700 + [0] * 90 + [1] * 20, [i % 50 for i in range(810)], 16, 1, 1, 32, "bfloat16", four, 16)
    run(dev, [700, 0, 3], [0, 0, 600], 16, 2, 1, 64, "bfloat16", four, 64)


@pytest.mark.parametrize("four", [False, True])
def test_strided_caches_and_rows(dev, four):
    """Heads before slots; keys and values in one buffer; rows of one projection."""
    run(dev, [3, 9], [1, 0], 4, 2, 3, 64, "bfloat16", four, 32, place=heads_first)
    page, Hkv, D = 4, 2, 16
    width = D // 2 + 4 if four else D
    fused = make((6, 3 * Hkv, D), "bfloat16", 1).to(dev)
    q, k, v = fused.split(Hkv, 1)
    kind = torch.uint8 if four else torch.bfloat16
    both = torch.zeros((5, 2, page, Hkv, width), dtype=kind, device=dev)
    kc, vc = (torch.zeros((5, page, Hkv, width), dtype=kind, device=dev) for _ in range(2))
    table = torch.tensor([[4, 0], [2, 3]], dtype=torch.int32, device=dev)
    off, starts = torch.tensor([0, 5, 6], device=dev), torch.tensor([1, 7], device=dev)
    t = angles(8, D).to(dev)
    a = OPS.paged_cache_append_rotary(q, k, v, off, starts, t, both[:, 0], both[:, 1], table)
    b = OPS.paged_cache_append_rotary(q.contiguous(), k.contiguous(), v.contiguous(), off, starts, t, kc, vc, table)
    assert torch.equal(a, b) and torch.equal(both[:, 0], kc) and torch.equal(both[:, 1], vc)
    assert torch.count_nonzero(kc) > 0


@pytest.mark.parametrize("four", [False, True])
def test_what_has_no_place_or_angle_is_dropped(dev, four):
    page, Hkv, D, R = 4, 1, 16, 8
    dtype = "float16"
    k, v, q = (make((12, Hkv, D), dtype, s) for s in (1, 2, 3))
    table = torch.tensor([[0, 1], [7, 2], [-1, 3], [1, 1]], dtype=torch.int32)
    off, starts = [1, 5, 7, 11, 11], [6, 3, 3, 0]
    t = angles(7, R)  # position 7 and further have no angle
    kc = torch.zeros((4, page, Hkv, D // 2 + 4 if four else D), dtype=torch.uint8 if four else DT[dtype])
    kd, vd = kc.to(dev), kc.to(dev)
    qr = OPS.paged_cache_append_rotary(q.to(dev), k.to(dev), v.to(dev), torch.tensor(off, device=dev),
                                       torch.tensor(starts, device=dev), t.to(dev), kd, vd, table.to(dev))
    kr = rotate(k, off, t, starts)
    want_k, want_v = kc.clone(), kc.clone()
    r = (lambda x: rows4(x)) if four else (lambda x: x.to(DT[dtype]))
    for row, p, slot in ((1, 1, 2), (6, 2, 0), (8, 3, 0), (9, 3, 1), (10, 3, 2)):
        want_k[p, slot], want_v[p, slot] = r(kr[row]), r(v[row].float())
    assert torch.equal(bits(kd), bits(want_k)) and torch.equal(bits(vd), bits(want_v))
    want = rotate(q, off, t, starts).to(DT[dtype])
    nan = torch.isnan(want)
    assert int(nan.sum()) == 3 * R and torch.equal(torch.isnan(qr.cpu()), nan)
    assert torch.equal(qr.cpu().masked_fill(nan, 0), want.masked_fill(nan, 0))
    # Negative starts, and starts past 32 bits.
    before = kd.clone()
    OPS.paged_cache_append_rotary(None, k.to(dev), v.to(dev), torch.tensor(off, device=dev),
                                  torch.tensor([-1, 2 ** 33, -2 ** 40, 0], device=dev), t.to(dev), kd, vd, table.to(dev))
    assert torch.equal(kd, before)


def test_four_bit_rows_are_the_codecs(dev):
    """Constant rows, one large value, values near fp16's ends, zeros: the rows are
    those of the 4-bit codec op, and read back as its inverse gives them."""
    D = 40
    x = make((10, 1, D), "float16", 1)
    x[0], x[1], x[2] = 0.0, 3.25, -0.0
    x[3] = x[3] * 6e-8
    x[4, 0, 7] = 60000.0
    x[5] = x[5] * 1e-5 + 1000.0
    x[6, 0, ::2], x[6, 0, 1::2] = 65504.0, -65504.0
    x[7] = torch.arange(D) / 16
    kc = torch.zeros((10, 1, 1, D // 2 + 4), dtype=torch.uint8, device=dev)
    vc = torch.zeros_like(kc)
    table = torch.arange(10, dtype=torch.int32, device=dev).view(10, 1)
    off = torch.arange(11, device=dev)
    OPS.paged_cache_append(x.to(dev), (-x).to(dev), off, torch.zeros(10, dtype=torch.int64, device=dev), kc, vc, table)
    for c, y in ((kc, x), (vc, -x)):
        want = torch.ops.fbgemm.HalfToFusedNBitRowwiseQuantizedSBHalf(y.view(10, D).to(dev), 4)
        assert torch.equal(c.view(10, -1), want)
        assert torch.equal(c.view(10, -1).cpu(), rows4(y).view(10, -1))
    k, v = OPS.paged_cache_gather(kc, vc, table, off, 10, torch.float16)
    assert torch.equal(k.view(10, D), torch.ops.fbgemm.FusedNBitRowwiseQuantizedSBHalfToHalf(kc.view(10, -1), 4))


@pytest.mark.parametrize("four,dtype", [(True, "float16"), (True, "bfloat16"), (False, "float16"), (False, "bfloat16")])
@pytest.mark.parametrize("D", [8, 24, 32, 40, 64, 72, 96, 128])
@pytest.mark.parametrize("page", [1, 5, 16])
def test_gather(dev, four, dtype, D, page):
    lengths = [3, 0, 33, 1, 16]
    table, pages = page_table(lengths, page)
    Hkv = 3
    if four:
        kc, vc = (rows4(make((pages, page, Hkv, D), torch.float32, s)) for s in (1, 2))
        kv, vv = (torch.from_numpy(values4(c)).float().to(DT[dtype]) for c in (kc, vc))
    else:
        kc, vc = (make((pages, page, Hkv, D), dtype, s) for s in (1, 2))
        kv, vv = kc, vc
    off = np.concatenate([[0], np.cumsum(lengths)]).astype(int)
    at = [(b, t) for b, n in enumerate(lengths) for t in range(n)]
    p, s = [int(table[b, t // page]) for b, t in at], [t % page for _, t in at]
    for index, place in ((torch.int32, lambda c: c), (torch.int64, heads_first)):
        k, v = OPS.paged_cache_gather(place(kc.to(dev)), place(vc.to(dev)), table.to(dev),
                                      torch.from_numpy(off).to(dev, index), len(at), DT[dtype])
        assert torch.equal(bits(k), bits(kv[p, s])) and torch.equal(bits(v), bits(vv[p, s]))


@pytest.mark.parametrize("four", [False, True])
def test_gather_of_rows_without_a_token(dev, four):
    """Rows behind the last list or before the first, pages that are none, lists
    longer than the table."""
    page, Hkv, D = 4, 1, 16
    kc = empty_cache(3, page, Hkv, D, "bfloat16", False, 1)
    if four:
        kc = rows4(kc.float())
    vals = torch.from_numpy(values4(kc)).float().bfloat16() if four else kc
    table = torch.tensor([[2, 5], [-1, 1], [0, 0]], dtype=torch.int32)
    off = [2, 8, 14, 23]
    k, v = OPS.paged_cache_gather(kc.to(dev), kc.to(dev), table.to(dev), torch.tensor(off, device=dev), 25)
    want = torch.zeros((25, Hkv, D), dtype=torch.bfloat16)
    want[2:6] = vals[2]
    want[12:14] = vals[1, :2]
    want[14:18], want[18:22] = vals[0], vals[0]
    assert torch.equal(k.cpu(), want) and torch.equal(v.cpu(), want)
    # Fewer rows than the offsets tell.
    k, _ = OPS.paged_cache_gather(kc.to(dev), kc.to(dev), table.to(dev), torch.tensor(off, device=dev), 5)
    assert torch.equal(k.cpu(), want[:5])


def test_past_4_gib(dev):
    """The last pages of caches whose offsets pass 32 bits, in both kinds."""
    page, Hkv, D = 64, 8, 128
    for four in (False, True):
        row = (D // 2 + 4) if four else 2 * D
        pages = (5 << 30) // (page * Hkv * row) + 1
        kc = torch.zeros((pages, page, Hkv, D // 2 + 4 if four else D), dtype=torch.uint8 if four else torch.bfloat16,
                         device=dev)
        vc = torch.zeros_like(kc)
        table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device=dev)
        n, t = 100, angles(100, D)
        k, v = make((n, Hkv, D), "bfloat16", 1), make((n, Hkv, D), "bfloat16", 2)
        off = torch.tensor([0, n], device=dev)
        OPS.paged_cache_append_rotary(None, k.to(dev), v.to(dev), off, torch.tensor([0], device=dev), t.to(dev), kc, vc,
                                      table)
        kr = rotate(k, [0, n], t)
        want = rows4(kr) if four else kr.bfloat16()
        assert torch.equal(kc[pages - 1].cpu(), want[:64]) and torch.equal(kc[pages - 2, :36].cpu(), want[64:])
        got, _ = OPS.paged_cache_gather(kc, vc, table, off, n, torch.bfloat16)
        assert torch.equal(got.cpu(), torch.from_numpy(values4(want)).float().bfloat16() if four else want)
        del kc, vc


def test_versions_and_gradients(dev):
    """Caches count appends; rotated queries never come back without their graph."""
    kc, vc = (torch.zeros((2, 4, 1, 12), dtype=torch.uint8, device=dev) for _ in range(2))
    k = make((1, 1, 16), "float16", 1).to(dev)
    off, starts = torch.tensor([0, 1], device=dev), torch.tensor([0], device=dev)
    t, table = angles(4, 16).to(dev), torch.tensor([[1]], dtype=torch.int32, device=dev)
    v0 = kc._version, vc._version
    OPS.paged_cache_append(k, k, off, starts, kc, vc, table)
    OPS.paged_cache_append_rotary(k, k, k, off, starts, t, kc, vc, table)
    assert (kc._version, vc._version) == (v0[0] + 2, v0[1] + 2)
    q = k.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        OPS.paged_cache_append_rotary(q, k, k, off, starts, t, kc, vc, table)
    with torch.no_grad():
        OPS.paged_cache_append_rotary(q, k, k, off, starts, t, kc, vc, table)
    with torch.inference_mode():
        inner = torch.zeros_like(kc)
        OPS.paged_cache_append_rotary(q, k, k, off, starts, t, inner, inner.clone(), table)
    assert torch.equal(inner, kc)


def test_empty(dev):
    for four in (False, True):
        w, kind = (20, torch.uint8) if four else (32, torch.float16)
        kc = torch.zeros((0, 16, 2, w), dtype=kind, device=dev)
        k = make((2, 2, 32), "float16", 0).to(dev)
        off, n, t = torch.tensor([0, 1, 2], device=dev), torch.tensor([5, 5], device=dev), angles(8, 32).to(dev)
        for W in (0, 3):
            table = torch.zeros((2, W), dtype=torch.int32, device=dev)
            q = OPS.paged_cache_append_rotary(k, k, k, off, n, t, kc, kc.clone(), table)
            assert torch.equal(q, OPS.jagged_rotary(k, off, t, n))
            OPS.paged_cache_append(k, k, off, n, kc, kc.clone(), table)
            a, b = OPS.paged_cache_gather(kc, kc, table, off, 2, torch.float16)
            assert a.shape == (2, 2, 32) and torch.count_nonzero(a) == 0 and torch.count_nonzero(b) == 0
        kc = torch.zeros((2, 16, 2, w), dtype=kind, device=dev)
        table, none = torch.zeros((0, 1), dtype=torch.int32, device=dev), torch.zeros(0, dtype=torch.int64, device=dev)
        zero = torch.tensor([0], device=dev)
        assert OPS.paged_cache_append_rotary(k[:0], k[:0], k[:0], zero, none, t, kc, kc.clone(), table).shape == (0, 2, 32)
        OPS.paged_cache_append(k[:0], k[:0], zero, none, kc, kc.clone(), table)
        assert OPS.paged_cache_gather(kc, kc, table, zero, 0, torch.float16)[0].shape == (0, 2, 32)
        assert torch.count_nonzero(OPS.paged_cache_append_rotary(k, k, k, zero, none, t, kc, kc.clone(), table)) == 0
        assert torch.count_nonzero(kc) == 0


def test_refusals(dev):
    kc = torch.zeros((2, 16, 2, 20), dtype=torch.uint8, device=dev)  # D 32
    h = torch.zeros((2, 16, 2, 32), dtype=torch.float16, device=dev)
    k = torch.zeros((4, 2, 32), dtype=torch.float16, device=dev)
    off, starts = torch.tensor([0, 1, 2, 4], device=dev), torch.ones(3, dtype=torch.int64, device=dev)
    table, t = torch.zeros((3, 1), dtype=torch.int32, device=dev), angles(8, 32).to(dev)
    wide = torch.zeros((2, 16, 2, 24), dtype=torch.uint8, device=dev)
    for args in [(k.float(), k.float(), off, starts, kc, kc, table), (k, k.bfloat16(), off, starts, kc, kc, table),
                 (k, k, off, starts, kc, h, table), (k, k, off, starts, wide, wide, table),
                 (k, k, off, starts, kc[..., :18], kc[..., :18], table), (k[:, :1], k[:, :1], off, starts, kc, kc, table),
                 (k, k, off, starts, kc[..., 1:], kc[..., 1:], table), (k, k, off, starts, kc.char(), kc.char(), table),
                 (k, k, off[:3], starts, kc, kc, table), (k, k, off, starts[:2], kc, kc, table),
                 (k, k, off, starts, kc.transpose(2, 3), kc.transpose(2, 3), table)]:
        with pytest.raises((RuntimeError, NotImplementedError)):
            OPS.paged_cache_append(*args)
    for args in [(k[:3], k, k, off, starts, t, kc, kc, table), (k.bfloat16(), k, k, off, starts, t, kc, kc, table),
                 (k[:, :, :16], k, k, off, starts, t, kc, kc, table), (k, k, k, off, starts, t.double(), kc, kc, table),
                 (k, k, k, off, starts, t[:, :3], kc, kc, table), (k, k, k, off, starts, t.cpu(), kc, kc, table),
                 (k, k, k, off, starts, angles(8, 40).to(dev), kc, kc, table), (k, k, k, off, starts, t[0], kc, kc, table),
                 (k, k.bfloat16(), k.bfloat16(), off, starts, t, h, h, table), (k, k, k, off, starts, t, kc, kc, table.long()),
                 (k, k, k, off, starts.float(), t, kc, kc, table), (k.cpu(), k, k, off, starts, t, kc, kc, table)]:
        with pytest.raises((RuntimeError, NotImplementedError)):
            OPS.paged_cache_append_rotary(*args)
    for args in [(kc, h, table, off, 4), (kc, kc, table, off, -1), (kc, kc, table, off[:3], 4),
                 (kc, kc, table, off, 4, torch.float32), (h, h, table, off, 4, torch.bfloat16),
                 (kc, kc, table.long(), off, 4), (kc, kc, table, off.float(), 4), (kc, kc, table, off.cpu(), 4),
                 (h.float(), h.float(), table, off, 4)]:
        with pytest.raises((RuntimeError, NotImplementedError)):
            OPS.paged_cache_gather(*args)

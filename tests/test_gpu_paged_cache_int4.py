"""Attention of one token per sequence over a cache of 4-bit rows, against its
float64 definition."""

import numpy as np
import pytest
import torch

from attention_helpers import check
from rows_helpers import attention4, make, page_table, rows4

pytestmark = pytest.mark.gpu

OPS = torch.ops.mx_fbgemm


def make_cache(lengths, page, Hkv, D, seed=0, fill=None, width=None, values=None):
    """Sequences' rows laid into pages in a random order.  Slots and pages of no token
    hold random bytes, their scale and bias `fill`."""
    table, pages = page_table(lengths, page, seed, width=width)
    g = torch.Generator().manual_seed(seed)
    caches, lists = [], []
    for which in range(2):
        c = torch.randint(0, 256, (pages, page, Hkv, D // 2 + 4), generator=g, dtype=torch.uint8)
        if fill is not None:
            c[..., -4:] = torch.full((2,), fill, dtype=torch.float16).view(torch.uint8)
        rows = []
        for b, n in enumerate(lengths):
            x = values(which, b, n) if values else make((n, Hkv, D), torch.float32, seed + 2 * b + which + 1)
            r = rows4(x) if n else torch.zeros((0, Hkv, D // 2 + 4), dtype=torch.uint8)
            rows.append(r)
            t = torch.arange(n)
            c[table[b, t // page].long(), t % page] = r
        caches.append(c), lists.append(rows)
    return caches[0], caches[1], table, lists[0], lists[1]


def run(dev, lengths, page, H, Hkv, D, dtype, index=torch.int32, scale=None, q=None, **kw):
    print(f"[case] {len(lengths)} lists up to {max(lengths)} page={page} H={H}/{Hkv} D={D} {dtype}", flush=True)
    kc, vc, table, ks, vs = make_cache(lengths, page, Hkv, D, **kw)
    if q is None:
        q = make((len(lengths), H, D), dtype, 99)
    out = OPS.paged_cache_attention(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev),
                                    torch.tensor(lengths, device=dev, dtype=index), scale)
    want, tol = attention4(q.double().numpy(), ks, vs, scale if scale is not None else D ** -0.5, dtype)
    check(out.double().cpu().numpy(), want, tol, "out")
    return out


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("D", [8, 16, 24, 32, 40, 48, 64, 72, 80, 96, 104, 120, 128])
def test_widths(dev, dtype, D):
    run(dev, [1, 0, 31, 32, 33, 200], 16, 4, 2, D, dtype)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("D", [8, 24, 32, 40, 64, 72, 96, 104, 128])
def test_widths_in_shares(dev, dtype, D):
    """More tokens than two wide blocks' tiles: sequences cut anywhere and joined."""
    run(dev, [1, 0, 31, 1300, 33, 129], 16, 4, 2, D, dtype)


@pytest.mark.parametrize("page", [1, 3, 8, 16, 33, 64, 100, 256])
def test_page_sizes(dev, page):
    run(dev, [1, 97, 300, 128], page, 4, 4, 64, "bfloat16", torch.int64)


@pytest.mark.parametrize("H,Hkv", [(1, 1), (2, 1), (16, 1), (17, 1), (40, 2), (24, 8)])
def test_grouped_heads(dev, H, Hkv):
    run(dev, [65, 5], 16, H, Hkv, 32, "float16", scale=0.3)


@pytest.mark.parametrize("B", [1, 3, 300])
def test_long_and_ragged(dev, B):
    rng = np.random.default_rng(B)
    lengths = [int(x) for x in rng.integers(0, 120, B)]
    lengths[0] = 5000 if B < 300 else 700
    run(dev, lengths, 16, 2, 1, 64, "bfloat16")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("room", [128, 144, 512, 528, 1024, 1040, 4096])
def test_room_in_the_table(dev, D, room):
    """The table's width decides how sequences are cut, not what comes out."""
    run(dev, [room - 1, 100, room // 2], 16, 6, 2, D, "float16")


@pytest.mark.parametrize("lengths", [[5, 50, 17], [5, 1490, 0, 17]])
@pytest.mark.parametrize("fill", [0.0, float("nan"), float("inf"), -float("inf")])
def test_what_slots_without_tokens_hold(dev, fill, lengths):
    run(dev, lengths, 100, 4, 2, 128, "bfloat16", fill=fill)
    run(dev, lengths, 100, 4, 2, 128, "float16", fill=fill)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_rows_far_from_zero(dev, dtype):
    """Biases that outweigh the codes, constant rows, small and large scales."""
    def values(which, b, n):
        x = make((n, 2, 64), torch.float32, 7 * b + which)
        return [x * 0.01 + 20.0, x * 0 + 3.0, x * 1e-4, x * 50][b]
    run(dev, [70, 40, 300, 33], 16, 4, 2, 64, dtype, values=values)


@pytest.mark.parametrize("size", [1e-30, 1e-6, 300.0, 3e4])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_sizes_of_queries(dev, dtype, size):
    """Queries far from order one; large ones make one token win."""
    q = (make((3, 4, 64), torch.float32, 5) * size).clamp(-65000, 65000).to(getattr(torch, dtype))
    run(dev, [70, 40, 300], 16, 4, 2, 64, dtype, q=q, scale=1.0 / max(size, 1e-6) if size > 1 else None)


def test_one_head_of_many_lists(dev):
    run(dev, [i % 130 for i in range(2100)], 16, 2, 1, 32, "bfloat16")


def test_lengths_past_the_table_and_below_zero(dev):
    kc, vc, table, ks, vs = make_cache([32, 32, 20], 16, 1, 32)
    q = make((3, 2, 32), "float16", 1).to(dev)
    args = (q, kc.to(dev), vc.to(dev), table.to(dev))
    want = OPS.paged_cache_attention(*args, torch.tensor([32, 32, 0], device=dev))
    got = OPS.paged_cache_attention(*args, torch.tensor([1000, 32, -7], device=dev))
    assert torch.equal(got, want) and torch.count_nonzero(got[2]) == 0


def test_bad_table_entries_are_absent_tokens(dev):
    kc, vc, table, ks, vs = make_cache([48, 48], 16, 1, 32)
    q = make((2, 2, 32), "float16", 1)
    lengths = torch.tensor([48, 48], device=dev)
    for bad in (-1, kc.size(0), 2 ** 31 - 1, -2 ** 31):
        t = table.clone()
        t[0, 1] = bad
        t[1] = bad
        out = OPS.paged_cache_attention(q.to(dev), kc.to(dev), vc.to(dev), t.to(dev), lengths)
        keep = [*range(16), *range(32, 48)]
        want, tol = attention4(q[:1].double().numpy(), [ks[0][keep]], [vs[0][keep]], 32 ** -0.5, "float16")
        check(out[:1].double().cpu().numpy(), want, tol, "out")
        assert torch.count_nonzero(out[1]) == 0


@pytest.mark.parametrize("D", [32, 64, 72, 128])
def test_strided_caches(dev, D):
    """Keys and values interleaved in one buffer, heads before slots, rows at any
    multiple of 4 bytes, tables and queries that are views: the same bits."""
    lengths = [70, 9]
    kc, vc, table, ks, vs = make_cache(lengths, 16, 2, D)
    q = make((2, 8, D), "bfloat16", 5).to(dev)
    n = torch.tensor(lengths, device=dev)
    table, kd, vd = table.to(dev), kc.to(dev), vc.to(dev)
    want = OPS.paged_cache_attention(q, kd, vd, table, n)
    both = torch.stack([kd, vd], 1)
    assert torch.equal(OPS.paged_cache_attention(q, both[:, 0], both[:, 1], table, n), want)
    hk, hv = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (kd, vd))
    assert torch.equal(OPS.paged_cache_attention(q, hk, hv, table, n), want)
    row = kd.size(3)
    for pad in (4, 12, 16):
        wk, wv = (torch.full((*x.shape[:3], row + pad), 255, dtype=torch.uint8, device=dev) for x in (kd, vd))
        wk[..., pad:], wv[..., :row] = kd, vd
        assert torch.equal(OPS.paged_cache_attention(q, wk[..., pad:], wv[..., :row], table, n), want)
    wide = torch.zeros((2, 5), dtype=torch.int32, device=dev)
    wide[:, : table.size(1)] = table
    assert torch.equal(OPS.paged_cache_attention(q, kd, vd, torch.cat([wide, wide], 1)[:, :5], n), want)
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(OPS.paged_cache_attention(qt, kd, vd, table, n), want)


def test_the_cache_ends_with_its_last_row(dev):
    """Rows at the very end of an allocation: nothing behind them is read into a
    result (the bytes behind are all ones, a NaN in scale and bias)."""
    for D in (8, 40, 72, 128):
        kc, vc, table, ks, vs = make_cache([16], 16, 1, D, width=1)
        row = D // 2 + 4
        pool = torch.full((kc.numel() + 4096,), 255, dtype=torch.uint8, device=dev)
        pool[: kc.numel()] = kc.reshape(-1).to(dev)
        view = pool[: kc.numel()].view(kc.shape)
        last = torch.tensor([[kc.size(0) - 1]], dtype=torch.int32, device=dev)
        view[-1] = kc[int(table[0, 0])].to(dev)
        q = make((1, 2, D), "bfloat16", 3)
        out = OPS.paged_cache_attention(q.to(dev), view, vc.to(dev)[int(table[0, 0])].expand(kc.shape).contiguous(), last,
                                        torch.tensor([16], device=dev))
        want, tol = attention4(q.double().numpy(), ks, vs, D ** -0.5, "bfloat16")
        check(out.double().cpu().numpy(), want, tol, f"out D={D} row={row}")


def test_the_same_bits_every_time(dev):
    kc, vc, table, ks, vs = make_cache([3000, 17, 900], 16, 2, 64)
    q = make((3, 4, 64), "float16", 1).to(dev)
    args = (q, kc.to(dev), vc.to(dev), table.to(dev), torch.tensor([3000, 17, 900], device=dev))
    want = OPS.paged_cache_attention(*args)
    for _ in range(5):
        assert torch.equal(OPS.paged_cache_attention(*args), want)


def test_empty(dev):
    kc = torch.zeros((0, 16, 2, 20), dtype=torch.uint8, device=dev)
    q = make((2, 2, 32), "float16", 0).to(dev)
    n = torch.tensor([5, 5], device=dev)
    for W in (0, 3):
        table = torch.zeros((2, W), dtype=torch.int32, device=dev)
        assert torch.count_nonzero(OPS.paged_cache_attention(q, kc, kc, table, n)) == 0
    kc = torch.zeros((2, 16, 2, 20), dtype=torch.uint8, device=dev)
    table = torch.zeros((0, 1), dtype=torch.int32, device=dev)
    assert OPS.paged_cache_attention(q[:0], kc, kc, table, n[:0]).shape == (0, 2, 32)


def test_refusals(dev):
    kc = torch.zeros((2, 16, 2, 20), dtype=torch.uint8, device=dev)  # D 32
    q = torch.zeros((3, 4, 32), dtype=torch.float16, device=dev)
    table = torch.zeros((3, 1), dtype=torch.int32, device=dev)
    n = torch.ones(3, dtype=torch.int64, device=dev)
    h = torch.zeros((2, 16, 2, 32), dtype=torch.float16, device=dev)
    big = torch.zeros((2, 16, 2, 72), dtype=torch.uint8, device=dev)
    for args in [(q.float(), kc, kc, table, n), (q[:, :3], kc, kc, table, n), (q[:, :, :16], kc, kc, table, n),
                 (q, kc[..., :18], kc[..., :18], table, n), (q, kc, kc[:1], table, n), (q, kc, h, table, n),
                 (q, kc[..., :4], kc[..., :4], table, n), (q, big, big, table, n), (q, kc.char(), kc.char(), table, n),
                 (q, kc.transpose(2, 3), kc.transpose(2, 3), table, n), (q, kc.cpu(), kc, table, n),
                 (q, kc, kc, table, n, 0.0), (q, kc, kc, table, n.float()), (q, kc[0], kc[0], table, n)]:
        with pytest.raises((RuntimeError, NotImplementedError)):
            OPS.paged_cache_attention(*args)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("lengths", [[90, 5], [2000, 33]])
def test_rows_of_very_different_sizes_in_one_sequence(dev, dtype, lengths):
    """Scales 2^-8 to 2^8 of each other among a sequence's values, the largest in the
    middle: p s keeps its bits whichever comes first, and small values are not lost
    where large ones get no weight."""
    def values(which, b, n):
        x = make((n, 2, 64), torch.float32, 3 * b + which)
        if which == 0:
            return x
        size = 2.0 ** (16 * torch.rand(n, generator=torch.Generator().manual_seed(b)) - 8)
        size[n // 2] = 2.0 ** 8
        return x * size[:, None, None]
    run(dev, lengths, 16, 4, 2, 64, dtype, values=values)
    run(dev, lengths, 16, 4, 2, 64, dtype, values=values, scale=4.0)


@pytest.mark.parametrize("dtype,large", [("float16", 60000.0), ("bfloat16", 1e20)])
def test_heads_of_very_different_sizes(dev, dtype, large):
    """A head whose queries do not fit beside its neighbours' (each has a power of two
    of its own); its one winning token, the others' ordinary weights."""
    q = make((2, 4, 64), torch.float32, 5)
    q[:, 1] *= large / 4
    q[:, 2] *= 1e-4
    run(dev, [70, 600], 16, 4, 2, 64, dtype, q=q.clamp(-65000, 65000).to(getattr(torch, dtype)) if dtype == "float16"
        else q.to(torch.bfloat16))


def test_wide_pages_and_pages_that_no_multiple_of_16_has(dev):
    """The same rows in pages of 16 (addresses by the wave) and of 24 (by the lanes):
    the same bits."""
    D, n = 128, [300, 77]
    outs = []
    rows = [[rows4(make((m, 2, D), torch.float32, 7 * w + m)) for m in n] for w in range(2)]
    q = make((2, 4, D), "bfloat16", 3).to(dev)
    for page in (16, 24, 48):
        table, pages = page_table(n, page, width=-(-320 // page))
        caches = [torch.zeros((pages, page, 2, D // 2 + 4), dtype=torch.uint8) for _ in range(2)]
        for c, lists in zip(caches, rows):
            for b, m in enumerate(n):
                t = torch.arange(m)
                c[table[b, t // page].long(), t % page] = lists[b]
        outs.append(OPS.paged_cache_attention(q, caches[0].to(dev), caches[1].to(dev), table.to(dev),
                                              torch.tensor(n, device=dev)))
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_page_strides_past_31_bits_are_refused(dev):
    """Strides are 32-bit numbers in the kernel: larger ones end at the host."""
    kc = torch.zeros(1 << 10, dtype=torch.uint8, device=dev).as_strided((1, 2, 1, 20), (1 << 31, 20, 20, 1))
    q = torch.zeros((1, 1, 32), dtype=torch.float16, device=dev)
    table, n = torch.zeros((1, 1), dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int64, device=dev)
    with pytest.raises(RuntimeError, match="2\\^31"):
        OPS.paged_cache_attention(q, kc, kc, table, n)
    kc = torch.zeros(1 << 10, dtype=torch.uint8, device=dev).as_strided((1, 1, 1, 20), (20, 1 << 31, 20, 1))
    with pytest.raises(RuntimeError, match="2\\^31"):
        OPS.paged_cache_attention(q, kc, kc, table, n)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lengths", [[70, 40], [3000, 40]])
@pytest.mark.parametrize("where", ["k", "v", "q"])
def test_nan_of_a_token_shows_in_its_sequence_alone(dev, D, lengths, where):
    for at in (0, 33, lengths[0] - 1):
        kc, vc, table, ks, vs = make_cache(lengths, 16, 2, D)
        q = make((2, 4, D), "bfloat16", 1)
        if where == "q":
            q[0, 1, 5] = float("nan")
        else:
            c = kc if where == "k" else vc
            c[int(table[0, at // 16]), at % 16, 0, -4:-2] = torch.tensor([float("nan")], dtype=torch.float16).view(torch.uint8)
        out = OPS.paged_cache_attention(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), torch.tensor(lengths, device=dev)).cpu()
        bad = torch.isnan(out[0]).all(-1)
        assert bad.tolist() == ([False, True, False, False] if where == "q" else [True, True, False, False]), at
        want, tol = attention4(q[1:].double().numpy(), ks[1:], vs[1:], D ** -0.5, "bfloat16")
        check(out[1:].double().numpy(), want, tol, "the other sequence")


@pytest.mark.parametrize("pattern", ["ragged", "empty first", "empty last", "one long", "alternating"])
def test_shares_over_more_sequences_than_lanes(dev, pattern):
    """Tables long enough for shares, sequences in several groups of 64: shares that
    begin or end before a sequence's first tile, and sequences without tokens
    wherever a share begins."""
    B, long = 170, 2300
    rng = np.random.default_rng(len(pattern))
    n = rng.integers(1, 400, B)
    if pattern == "empty first":
        n[:70] = 0
    elif pattern == "empty last":
        n[-75:] = 0
    elif pattern == "one long":
        n[:] = 1
    elif pattern == "alternating":
        n[::2] = 0
    n[100 if pattern != "empty last" else 20] = long
    run(dev, [int(x) for x in n], 16, 2, 1, 32, "float16")


@pytest.mark.parametrize("pattern", ["ragged", "ones", "empty around"])
def test_shares_of_many_heads(dev, pattern):
    """Fewer workers than sequences, and shares of a unit each."""
    n = {"ragged": [1, 1500, 3, 0, 1100, 129, 128, 127], "ones": [1, 1, 1, 1],
         "empty around": [0, 0, 1200, 0, 0, 7, 0]}[pattern]
    run(dev, n, 16, 16, 8, 64, "bfloat16")
    kc, vc, table, ks, vs = make_cache(n, 16, 8, 64, width=160)
    q = make((len(n), 16, 64), "bfloat16", 3)
    out = OPS.paged_cache_attention(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), torch.tensor(n, device=dev))
    want, tol = attention4(q.double().numpy(), ks, vs, 64 ** -0.5, "bfloat16")
    check(out.double().cpu().numpy(), want, tol, "out")

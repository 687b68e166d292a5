"""The paged key-value cache on the GPU: appends bit for bit, attention of one
token per sequence against its float64 definition, and their refusals."""

import numpy as np
import pytest
import torch

from attention_helpers import check, paged_attention

pytestmark = pytest.mark.gpu

DT = {"float16": torch.float16, "bfloat16": torch.bfloat16}
OPS = torch.ops.mx_fbgemm


def make(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(DT[dtype])


def make_cache(lengths, page, Hkv, D, dtype, seed=0, fill=float("nan"), extra=3):
    """Per-sequence keys and values laid into pages in a random order; slots and
    pages of no token hold `fill`, table entries of no page -1."""
    rng = np.random.default_rng(seed)
    need = [-(-n // page) for n in lengths]
    width = max(need + [1])
    order = rng.permutation(sum(need) + extra)
    table = np.full((len(lengths), width), -1, np.int32)
    kc = torch.full((order.size, page, Hkv, D), fill, dtype=DT[dtype])
    vc = kc.clone()
    ks, vs, at = [], [], 0
    for b, n in enumerate(lengths):
        table[b, : need[b]] = order[at: at + need[b]]
        at += need[b]
        k, v = make((n, Hkv, D), dtype, seed + 2 * b + 1), make((n, Hkv, D), dtype, seed + 2 * b + 2)
        ks.append(k), vs.append(v)
        for t in range(n):
            kc[table[b, t // page], t % page] = k[t]
            vc[table[b, t // page], t % page] = v[t]
    return kc, vc, torch.from_numpy(table), ks, vs


def run(dev, lengths, page, H, Hkv, D, dtype, index=torch.int32, scale=None, **kw):
    print(f"[case] lengths={lengths} page={page} H={H}/{Hkv} D={D} {dtype}", flush=True)
    kc, vc, table, ks, vs = make_cache(lengths, page, Hkv, D, dtype, **kw)
    q = make((len(lengths), H, D), dtype, 99)
    out = OPS.paged_cache_attention(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev),
                                    torch.tensor(lengths, device=dev, dtype=index), scale)
    want, tol = paged_attention(q.double().numpy(), [k.double().numpy() for k in ks],
                                [v.double().numpy() for v in vs],
                                scale if scale is not None else D ** -0.5, dtype)
    check(out.double().cpu().numpy(), want, tol, "out")
    return out


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("D", [8, 32, 40, 64, 72, 96, 104, 128])
def test_widths(dev, dtype, D):
    run(dev, [1, 0, 31, 32, 33, 200], 16, 4, 2, D, dtype)


@pytest.mark.parametrize("page", [1, 3, 8, 16, 33, 64, 100, 256])
def test_page_sizes(dev, page):
    """Pages that end inside a tile, and tiles inside a page."""
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


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("D", [8, 32, 40, 64, 72, 96, 104, 128])
def test_widths_in_shares(dev, dtype, D):
    """More tokens than two wide blocks' tiles: sequences cut anywhere and joined."""
    run(dev, [1, 0, 31, 1300, 33, 129], 16, 4, 2, D, dtype)


@pytest.mark.parametrize("fill", [0.0, float("nan"), float("inf"), -float("inf")])
def test_what_slots_in_shares_hold(dev, fill):
    run(dev, [5, 1490, 0, 17], 100, 4, 2, 64, "bfloat16", fill=fill)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("room", [128, 144, 512, 528, 1024, 1040, 4096])
def test_room_in_the_table(dev, D, room):
    """The table's width decides how sequences are cut, not what comes out."""
    kc, vc, table, ks, vs = make_cache([room - 1, 100, room // 2], 16, 2, D, "bfloat16")
    q = make((3, 6, D), "bfloat16", 9)
    out = OPS.paged_cache_attention(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev),
                                    torch.tensor([room - 1, 100, room // 2], device=dev))
    want, tol = paged_attention(q.double().numpy(), [k.double().numpy() for k in ks],
                                [v.double().numpy() for v in vs], D ** -0.5, "bfloat16")
    check(out.double().cpu().numpy(), want, tol, "out")


@pytest.mark.parametrize("fill", [0.0, float("nan"), float("inf"), -float("inf")])
def test_what_slots_without_tokens_hold(dev, fill):
    run(dev, [5, 50, 17], 16, 4, 2, 128, "bfloat16", fill=fill)


def test_lengths_past_the_table_and_below_zero(dev):
    kc, vc, table, ks, vs = make_cache([32, 32, 20], 16, 1, 32, "float16")
    q = make((3, 2, 32), "float16", 1).to(dev)
    args = (q, kc.to(dev), vc.to(dev), table.to(dev))
    want = OPS.paged_cache_attention(*args, torch.tensor([32, 32, 0], device=dev))
    got = OPS.paged_cache_attention(*args, torch.tensor([1000, 32, -7], device=dev))
    assert torch.equal(got, want) and torch.count_nonzero(got[2]) == 0


def test_bad_table_entries_are_absent_tokens(dev):
    """An entry outside the cache's pages hides its tokens, whatever it is."""
    kc, vc, table, ks, vs = make_cache([48, 48], 16, 1, 32, "float16")
    q = make((2, 2, 32), "float16", 1)
    lengths = torch.tensor([48, 48], device=dev)
    for bad in (-1, kc.size(0), 2 ** 31 - 1, -2 ** 31):
        t = table.clone()
        t[0, 1] = bad
        t[1] = bad
        out = OPS.paged_cache_attention(q.to(dev), kc.to(dev), vc.to(dev), t.to(dev), lengths)
        keep = [*range(16), *range(32, 48)]
        want, tol = paged_attention(q[:1].double().numpy(), [ks[0][keep].double().numpy()],
                                    [vs[0][keep].double().numpy()], 32 ** -0.5, "float16")
        check(out[:1].double().cpu().numpy(), want, tol, "out")
        assert torch.count_nonzero(out[1]) == 0


def test_strided_caches(dev):
    """Keys and values interleaved in one buffer, and heads before slots."""
    lengths = [70, 9]
    kc, vc, table, ks, vs = make_cache(lengths, 16, 2, 64, "bfloat16", fill=0.0)
    q = make((2, 8, 64), "bfloat16", 5).to(dev)
    n = torch.tensor(lengths, device=dev)
    table, kd, vd = table.to(dev), kc.to(dev), vc.to(dev)
    want = OPS.paged_cache_attention(q, kd, vd, table, n)
    both = torch.stack([kd, vd], 1)
    assert torch.equal(OPS.paged_cache_attention(q, both[:, 0], both[:, 1], table, n), want)
    hk, hv = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (kd, vd))
    assert torch.equal(OPS.paged_cache_attention(q, hk, hv, table, n), want)
    wide = torch.zeros((2, 5), dtype=torch.int32, device=dev)
    wide[:, : table.size(1)] = table
    wt = torch.cat([wide, wide], 1)[:, :5]
    assert torch.equal(OPS.paged_cache_attention(q, kd, vd, wt, n), want)
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(OPS.paged_cache_attention(qt, kd, vd, table, n), want)


@pytest.mark.parametrize("lists", [4, 200])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("page", [1, 5, 16])
def test_append(dev, lists, index, page):
    """Rows land where the table says, bit for bit; nothing else changes."""
    rng = np.random.default_rng(lists + page)
    n = rng.integers(0, 9, lists)
    starts = rng.integers(0, 40, lists)
    Hkv, D = 3, 40
    need = [-(-int(a + b) // page) for a, b in zip(n, starts)]
    order = rng.permutation(sum(need) + 2).astype(np.int32)
    table = np.full((lists, max(need + [1])), -1, np.int32)
    at = 0
    for b in range(lists):
        table[b, : need[b]] = order[at: at + need[b]]
        at += need[b]
    off = np.concatenate([[0], np.cumsum(n)])
    k, v = make((int(off[-1]), Hkv, D), "bfloat16", 1), make((int(off[-1]), Hkv, D), "bfloat16", 2)
    kc, vc = make((order.size, page, Hkv, D), "bfloat16", 3), make((order.size, page, Hkv, D), "bfloat16", 4)
    ke, ve = kc.clone(), vc.clone()
    for b in range(lists):
        for j in range(int(n[b])):
            t = int(starts[b]) + j
            ke[table[b, t // page], t % page] = k[off[b] + j]
            ve[table[b, t // page], t % page] = v[off[b] + j]
    kd, vd = kc.to(dev), vc.to(dev)
    OPS.paged_cache_append(k.to(dev), v.to(dev), torch.from_numpy(off).to(dev, index),
                           torch.from_numpy(starts).to(dev, index), kd, vd, torch.from_numpy(table).to(dev))
    assert torch.equal(kd.cpu().view(torch.int16), ke.view(torch.int16))
    assert torch.equal(vd.cpu().view(torch.int16), ve.view(torch.int16))


def test_append_drops_what_has_no_place(dev):
    """Rows of no list, tokens past the table, entries of no page."""
    page, Hkv, D = 4, 1, 8
    k, v = make((12, Hkv, D), "float16", 1), make((12, Hkv, D), "float16", 2)
    table = torch.tensor([[0, 1], [7, 2], [-1, 3], [1, 1]], dtype=torch.int32)
    off = torch.tensor([1, 5, 7, 11, 11])
    starts = torch.tensor([6, 3, 3, 0])
    kc, vc = torch.zeros((4, page, Hkv, D), dtype=torch.float16), torch.zeros((4, page, Hkv, D), dtype=torch.float16)
    kd, vd = kc.to(dev), vc.to(dev)
    OPS.paged_cache_append(k.to(dev), v.to(dev), off.to(dev), starts.to(dev), kd, vd, table.to(dev))
    for c, x in ((kc, k), (vc, v)):
        c[1, 2], c[1, 3] = x[1], x[2]          # list 0: tokens 6, 7; 8 and 9 past its row
        c[2, 0] = x[6]                         # list 1: token 3 on page 7 (none), token 4
        c[3, 0:3] = x[8:11]                    # list 2: token 3 on page -1, tokens 4..6
    assert torch.equal(kd.cpu(), kc) and torch.equal(vd.cpu(), vc)


def test_append_into_strided_caches_from_views(dev):
    page, Hkv, D = 4, 2, 16
    fused = make((6, 3 * Hkv, D), "bfloat16", 1).to(dev)
    k, v = fused[:, Hkv:2 * Hkv], fused[:, 2 * Hkv:]
    both = torch.zeros((5, 2, page, Hkv, D), dtype=torch.bfloat16, device=dev)
    table = torch.tensor([[4, 0], [2, 3]], dtype=torch.int32, device=dev)
    off, starts = torch.tensor([0, 5, 6], device=dev), torch.tensor([1, 7], device=dev)
    OPS.paged_cache_append(k, v, off, starts, both[:, 0], both[:, 1], table)
    want = torch.zeros_like(both)
    for i, x in enumerate((k, v)):
        for j in range(5):
            want[[4, 0][(1 + j) // 4], i, (1 + j) % 4] = x[j]
        want[3, i, 3] = x[5]
    assert torch.equal(both, want)


def test_cache_past_4_gib(dev):
    """Offsets past 32 bits, in bytes and in elements: the last pages of a large cache."""
    page, Hkv, D = 64, 8, 128
    pages = (5 << 30) // (page * Hkv * D * 2) + 1
    kc = torch.zeros((pages, page, Hkv, D), dtype=torch.bfloat16, device=dev)
    vc = torch.zeros_like(kc)
    n = 100
    k, v = make((n, Hkv, D), "bfloat16", 1), make((n, Hkv, D), "bfloat16", 2)
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device=dev)
    OPS.paged_cache_append(k.to(dev), v.to(dev), torch.tensor([0, n], device=dev),
                           torch.tensor([0], device=dev), kc, vc, table)
    assert torch.equal(kc[pages - 1].cpu(), k[:64]) and torch.equal(vc[pages - 2, :36].cpu(), v[64:])
    q = make((1, Hkv, D), "bfloat16", 3)
    out = OPS.paged_cache_attention(q.to(dev), kc, vc, table, torch.tensor([n], device=dev))
    want, tol = paged_attention(q.double().numpy(), [k.double().numpy()], [v.double().numpy()], D ** -0.5,
                                "bfloat16")
    check(out.double().cpu().numpy(), want, tol, "out")


def test_empty(dev):
    kc = torch.zeros((0, 16, 2, 32), dtype=torch.float16, device=dev)
    q = make((2, 2, 32), "float16", 0).to(dev)
    n = torch.tensor([5, 5], device=dev)
    for W in (0, 3):
        table = torch.zeros((2, W), dtype=torch.int32, device=dev)
        assert torch.count_nonzero(OPS.paged_cache_attention(q, kc, kc, table, n)) == 0
        OPS.paged_cache_append(q, q, torch.tensor([0, 1, 2], device=dev), n, kc, kc.clone(), table)
    kc = torch.zeros((2, 16, 2, 32), dtype=torch.float16, device=dev)
    table = torch.zeros((0, 1), dtype=torch.int32, device=dev)
    none = torch.zeros(0, dtype=torch.int64, device=dev)
    assert OPS.paged_cache_attention(q[:0], kc, kc, table, none).shape == (0, 2, 32)
    OPS.paged_cache_append(q[:0], q[:0], torch.tensor([0], device=dev), none, kc, kc.clone(), table)


def test_refusals(dev):
    kc = torch.zeros((2, 16, 2, 32), dtype=torch.float16, device=dev)
    vc = torch.zeros_like(kc)
    q = torch.zeros((3, 4, 32), dtype=torch.float16, device=dev)
    table = torch.zeros((3, 1), dtype=torch.int32, device=dev)
    n = torch.ones(3, dtype=torch.int64, device=dev)
    for args in [(q.float(), kc, vc, table, n), (q.bfloat16(), kc, vc, table, n),
                 (q.float(), kc.float(), vc.float(), table, n),
                 (q[:, :3], kc, vc, table, n), (q[:, :, :16], kc, vc, table, n),
                 (q[:2], kc, vc, table, n), (q, kc, vc, table, n[:2]),
                 (q, kc, vc, table.long(), n), (q, kc, vc, table.view(-1), n),
                 (q, kc, vc, table, n.float()), (q, kc, vc, table.cpu(), n), (q, kc, vc, table, n.cpu()),
                 (q, kc, vc[:1], table, n), (q, kc[0], vc[0], table, n),
                 (q, kc.transpose(2, 3), vc.transpose(2, 3), table, n),
                 (q, kc, vc, table, n, 0.0), (q, kc, vc, table, n, float("inf"))]:
        with pytest.raises((RuntimeError, NotImplementedError)):
            OPS.paged_cache_attention(*args)
    k = torch.zeros((4, 2, 32), dtype=torch.float16, device=dev)
    off, starts = torch.tensor([0, 1, 2, 4], device=dev), n
    for args in [(k.bfloat16(), k, off, starts, kc, vc, table), (k[:3], k, off, starts, kc, vc, table),
                 (k[:, :1], k[:, :1], off, starts, kc, vc, table), (k, k, off[:3], starts, kc, vc, table),
                 (k, k, off, starts[:2], kc, vc, table), (k, k, off.float(), starts, kc, vc, table),
                 (k, k, off, starts, kc.cpu(), vc, table), (k, k, off, starts, kc, vc, table.long())]:
        with pytest.raises((RuntimeError, NotImplementedError)):
            OPS.paged_cache_append(*args)

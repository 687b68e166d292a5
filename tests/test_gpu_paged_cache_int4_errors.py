"""Attention over 4-bit rows where a bound on single outputs says little: mean
square errors, every token counted once, scores and queries to their last bit."""

import numpy as np
import pytest
import torch

from attention_helpers import TINY, U
from int4_errors import attention4_errors, mean_square
from rows_helpers import make, page_table, rows4

pytestmark = pytest.mark.gpu

OPS = torch.ops.mx_fbgemm
LIMIT = 1.3  # as the planted mistakes of test_int4_errors.py have it


def raw_rows(codes, scale, bias):
    """Rows [..., D / 2 + 4] of given codes, scale and bias (both fp16)."""
    c = codes.to(torch.uint8)
    ends = torch.tensor([scale, bias], dtype=torch.float16).view(torch.uint8).expand(*c.shape[:-1], 4)
    return torch.cat([c[..., 0::2] | (c[..., 1::2] << 4), ends], -1)


def attend(dev, keys, values, q, page=16, scale=None, index=torch.int32):
    """keys, values: lists of rows [n, Hkv, D / 2 + 4], laid into pages in a random order."""
    lengths = [k.shape[0] for k in keys]
    table, pages = page_table(lengths, page, len(lengths))
    caches = []
    for lists in (keys, values):
        c = torch.randint(0, 256, (pages, page, *lists[0].shape[1:]), dtype=torch.uint8,
                          generator=torch.Generator().manual_seed(pages))
        for b, r in enumerate(lists):
            t = torch.arange(r.shape[0])
            c[table[b, t // page].long(), t % page] = r
        caches.append(c.to(dev))
    return OPS.paged_cache_attention(q.to(dev), *caches, table.to(dev), torch.tensor(lengths, device=dev, dtype=index),
                                     scale).double().cpu().numpy()


# Shares over long tables, blocks of their own, wide blocks, a wave's odd ends.
LENGTHS = {"long": [5000], "long and short": [3000, 1, 40, 0, 700], "blocks": [300, 1000, 128, 33] * 40, "wide": [900, 31]}


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("D", [32, 40, 64, 128])
@pytest.mark.parametrize("lists", list(LENGTHS))
@pytest.mark.parametrize("kind", ["plain", "mean", "outliers", "large keys"])
def test_mean_square_errors(dev, dtype, D, lists, kind):
    lengths = LENGTHS[lists]
    if lists == "blocks" and (kind != "plain" or D == 40):
        lengths = lengths[:8]
    print(f"[case] {lists} D={D} {dtype} {kind}", flush=True)
    Hkv = 2
    H = max(Hkv, -(-4096 // (D * sum(n > 0 for n in lengths) * Hkv)) * Hkv)  # 4,096 outputs or more
    q = make((len(lengths), H, D), torch.float32, 1)
    keys, values = ([make((n, Hkv, D), torch.float32, s + 2 * b) for b, n in enumerate(lengths)] for s in (3, 4))
    if kind == "mean":
        q += 1
    elif kind == "outliers":
        q[..., 1:D:D // 4] *= 10
        for k in keys:
            k[..., 1:D:D // 4] *= 20
    elif kind == "large keys":  # (a score's two parts outweigh it)
        keys = [k + 4 for k in keys]
    q = q.to(getattr(torch, dtype))
    keys, values = ([rows4(x) if x.shape[0] else torch.zeros((0, Hkv, D // 2 + 4), dtype=torch.uint8) for x in y]
                    for y in (keys, values))
    scale = D ** -0.5 if kind != "outliers" else 0.1 * D ** -0.5
    got = attend(dev, keys, values, q, scale=scale)
    want, var = attention4_errors(q.double().numpy(), keys, values, scale, dtype)
    some = np.array([n > 0 for n in lengths])
    off = mean_square(got[some], want[some], var[some])
    print(f"mean square {off:.3f}", flush=True)
    assert off <= LIMIT and (got[~some] == 0).all()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("D,lengths", [(32, [5000]), (64, [5000, 31, 1]), (128, [3001, 128, 129, 700]), (64, [1000, 900]),
                                       (128, [260] * 40), (64, [9000])])
def test_every_token_counts_once(dev, dtype, page, D, lengths):
    """Equal weights (queries of zeros), token j's value one in column j mod D: an output
    is a whole number of tokens over their number, rounded in fp32 and once more."""
    rng = torch.Generator().manual_seed(1)
    keys = [torch.randint(0, 256, (n, 1, D // 2 + 4), generator=rng, dtype=torch.uint8) for n in lengths]
    for k in keys:
        k[..., -4:] = torch.tensor([0.5, -3.0], dtype=torch.float16).view(torch.uint8)
    values, want = [], np.zeros((len(lengths), 2, D))
    for b, n in enumerate(lengths):
        codes = torch.full((n, 1, D), 8)
        codes[torch.arange(n), 0, torch.arange(n) % D] = 9
        values.append(raw_rows(codes, 1.0, -8.0))
        want[b] = np.bincount(np.arange(n) % D, minlength=D) / n
    got = attend(dev, keys, values, torch.zeros((len(lengths), 2, D), dtype=getattr(torch, dtype)), page)
    tol = want * (U[dtype] + 2.0 ** -22) + TINY[dtype]
    assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("n,B", [(2000, 64), (1100, 200), (300, 150)])
def test_the_one_token_that_counts(dev, dtype, n, B):
    """Sequences alike but for the place of the one token whose value is not zero: places
    over all seams of waves, tiles, pages and shares."""
    D = 32
    places = [(b * 131 + b // 8) % n for b in range(B)]
    places[:8] = [0, 31, 32, 127, 128, n - 1, n // 2, 1023 % n]
    keys = [raw_rows(torch.full((n, 1, D), 3), 0.5, 1.0)] * B
    values, want = [], np.zeros((B, 1, D))
    for b, at in enumerate(places):
        codes = torch.full((n, 1, D), 8)
        codes[at] = torch.arange(D) % 16
        values.append(raw_rows(codes, 1.0, -8.0))
        want[b] = (np.arange(D) % 16 - 8) / n
    got = attend(dev, keys, values, make((B, 1, D), dtype, 1))
    # Equal rows have equal scores; each tile's difference from the maximum is rounded
    # to fp32 once: 2^-24 of scores of up to 2^5 in base 2, twice.
    tol = np.abs(want) * (U[dtype] + 2.0 ** -17) + TINY[dtype]
    if dtype == "bfloat16":
        tol += np.abs(want) * 2.0 ** -11  # p s in fp16
    assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("D", [8, 32, 40, 64, 128])
@pytest.mark.parametrize("n", [2, 32, 1500])
def test_equal_scores_weigh_alike(dev, dtype, D, n):
    """A row's codes in another order against equal queries: sums of (c - 8) q are whole
    numbers below 2^24 in any order, so the scores are one number, and values of +1
    and -1 in turn leave zero.  (2^-15: the score's own rounding, of up to 2^-17 of a
    weight, beside the maximum of an earlier tile; in pairs it leaves zero too, but for the part
    that fp16 outputs' second operand rounds.)"""
    g = torch.Generator().manual_seed(D)
    row = torch.randint(0, 16, (D,), generator=g)
    keys = raw_rows(torch.stack([row[torch.randperm(D, generator=g)] for _ in range(n)])[:, None], 1.0, -8.0)
    signs = torch.where(torch.arange(n) % 2 == 0, 9, 7)
    values = raw_rows(signs[:, None, None].expand(n, 1, D), 1.0, -8.0)
    size = 2001.0 if dtype == "float16" else 2000.0  # 11 and 8 bits
    q = torch.full((1, 2, D), size).to(getattr(torch, dtype))
    got = attend(dev, [keys], [values], q, scale=1.0 / 2000)
    assert np.abs(got).max() <= 2.0 ** -15


@pytest.mark.parametrize("dtype,small", [("float16", 2.0 ** -11), ("bfloat16", 2.0 ** -15)])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("n", [2, 64, 1500])
def test_small_queries_beside_a_large_one(dev, dtype, small, D, n):
    """Queries of all their type's bits, 2^7 and 2^11 below the head's largest, against
    codes in even columns for one half of the tokens and in the odd ones (whose
    queries are alike) for the other: sums of multiples of q's last bit, below 2^24 of
    it, so scores are equal and values of +1 and -1 leave zero (to 2^-15, as above)."""
    g = torch.Generator().manual_seed(D)
    bits = 10 if dtype == "float16" else 7
    m = small * (1 + (2 * torch.randint(0, 2 ** (bits - 1), (D // 2,), generator=g) + 1) / 2 ** bits)
    q = m.repeat_interleave(2)
    q[:2] = 2.0 ** -4
    q = q.to(getattr(torch, dtype)).expand(1, 2, D).contiguous()
    codes = torch.randint(0, 16, (D // 2,), generator=g)
    codes[0] = 8
    even, odd = torch.full((2, D), 8).unbind(0)
    even[0::2], odd[1::2] = codes, codes
    keys = raw_rows(torch.stack([even, odd] * (n // 2))[:, None], 1.0, -8.0)
    signs = torch.where(torch.arange(n) % 2 == 0, 9, 7)
    values = raw_rows(signs[:, None, None].expand(n, 1, D), 1.0, -8.0)
    got = attend(dev, [keys], [values], q, scale=20.0 / (small * D ** 0.5))
    assert np.abs(got).max() <= 2.0 ** -15

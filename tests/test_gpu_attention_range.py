"""fp16 gradients whose dS = p (dO.v - delta) passes fp16's range while the gradients
themselves do not: loss-scaled training with a small softmax scale.

dS is rounded to 11 bits for a matrix product.  Where a column of it (a query's row for
dQ, a key's for dK) passes 65504, it is rounded at a power of two f that brings the
column's largest below 2^15, that is, 1 / f <= top 2^-14.  Beyond the bounds of
attention_helpers (which hold for normal values, and 2^-25 for subnormal ones), an
element can then be off by 2^-25 / f <= top 2^-39."""

import numpy as np
import pytest
import torch

from attention_helpers import attention, check, visible

pytestmark = pytest.mark.gpu

OPS = torch.ops.mx_fbgemm
MOST = 65504.0


def offsets_of(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)


def make(rows, heads, D, seed, scale):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((rows, heads, D), generator=g) * scale).clamp(-6e4, 6e4).half()


def fitted_extra(q, k, v, g, qo, ko, causal, scale):
    """What the columns' factors add to the bounds of dQ and dK, and the largest |dS|."""
    H, Hkv = q.shape[1], k.shape[1]
    G = H // Hkv
    dq, dk, largest = np.zeros_like(q), np.zeros_like(k), 0.0
    for b in range(len(qo) - 1):
        rq, rk = slice(qo[b], qo[b + 1]), slice(ko[b], ko[b + 1])
        nq, nk = rq.stop - rq.start, rk.stop - rk.start
        if nq == 0 or nk == 0:
            continue
        see = visible(nq, nk, causal)
        for h in range(Hkv):
            column = np.zeros(nk)
            for e in range(h * G, (h + 1) * G):
                s = np.where(see, q[rq, e] @ k[rk, h].T * scale, -np.inf)
                w = np.exp(s - np.where(see.any(1), s.max(1), 0.0)[:, None])
                w /= np.maximum(w.sum(1), 1e-300)[:, None]
                dw = g[rq, e] @ v[rk, h].T
                ds = np.abs(w * (dw - (w * dw).sum(1)[:, None]))
                largest = max(largest, ds.max())
                dq[rq, e] = scale * 2.0 ** -39 * (see * ds.max(1)[:, None]) @ np.abs(k[rk, h])
                column = np.maximum(column, ds.max(0))
            for e in range(h * G, (h + 1) * G):
                dk[rk, h] += scale * 2.0 ** -39 * (see * column[None, :]).T @ np.abs(q[rq, e])
    return dq, dk, largest


def run(dev, q, k, v, g, qo, ko, causal, scale, past_range=True):
    print(f"[case] q {tuple(q.shape)} k {tuple(k.shape)} causal={causal} lists={len(qo) - 1}", flush=True)
    x = [t.double().numpy() for t in (q, k, v)]
    want = attention(*x, qo, ko, causal, scale, "float16", g.double().numpy())
    more_q, more_k, largest = fitted_extra(*x, g.double().numpy(), qo, ko, causal, scale)
    assert (largest > MOST) == past_range
    for w in (want.out, want.dq, want.dk, want.dv):
        assert np.abs(w).max() < MOST
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v)]
    to, tk = (torch.from_numpy(o).to(dev) for o in (qo, ko))
    out = OPS.jagged_attention(*leaves, to, tk, causal, scale)
    got = torch.autograd.grad(out, leaves, g.to(dev))
    again = torch.autograd.grad(OPS.jagged_attention(*leaves, to, tk, causal, scale), leaves, g.to(dev))
    for name, y, z, w, tol in zip(("dq", "dk", "dv"), got, again, (want.dq, want.dk, want.dv),
                                  (want.dq_tol + 1.01 * more_q, want.dk_tol + 1.01 * more_k, want.dv_tol)):
        check(y.double().cpu().numpy(), w, tol, name)
        assert torch.equal(y, z)
    return got


# Lists, heads and widths that reach the launches with one and two groups of waves,
# heads packed into a block, and a key's queries in shares.
SHAPES = [([3, 1, 40, 64, 130], [3, 1, 40, 64, 130], 2, 2, 128), ([1500, 777], [1500, 777], 4, 1, 64),
          ([900, 300], [900, 300], 2, 1, 128), ([40, 7, 33, 90], [90, 300, 33, 20], 4, 2, 96),
          ([20, 0, 55], [20, 9, 500], 4, 1, 40), ([17, 70], [17, 70], 1, 1, 8)]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_scores_and_gradients_past_the_range_between(dev, shape, causal):
    nq, nk, H, Hkv, D = SHAPES[shape]
    qo, ko = offsets_of(nq), offsets_of(nk)
    scale = 0.000125 * (128 / D) ** 0.5
    q, k = make(qo[-1], H, D, 1, 37.6), make(ko[-1], Hkv, D, 2, 37.6)
    v, g = make(ko[-1], Hkv, D, 3, 18.0 * (128 / D) ** 0.5), make(qo[-1], H, D, 4, 5e3)
    run(dev, q, k, v, g, qo, ko, causal, scale)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,Hkv,D,n", [(2, 2, 128, 90), (4, 1, 64, 1100)])
def test_the_largest_values_of_the_type(dev, H, Hkv, D, n, causal):
    """dO and v of thousands to 6e4: dS of 1e8, brought back by the scale."""
    o = offsets_of([n, 5])
    q, k = make(o[-1], H, D, 1, 1.0), make(o[-1], Hkv, D, 2, 1.0)
    v, g = make(o[-1], Hkv, D, 3, 1e4), make(o[-1], H, D, 4, 4e3)
    run(dev, q, k, v, g, o, o, causal, 1e-7)


@pytest.mark.parametrize("causal", [True, False])
def test_large_rows_among_small_ones(dev, causal):
    """One query's gradients and one key's value are large, early, late or in between:
    a factor of its column alone, taken where the column passes the range."""
    n, D = 300, 64
    o = offsets_of([n])
    for at in (2, 150, n - 1):
        q, k = make(n, 1, D, 1, 53.0), make(n, 1, D, 2, 53.0)
        v, g = make(n, 1, D, 3, 1.0), make(n, 1, D, 4, 0.1)
        g[at] = make(1, 1, D, 5, 1.5e4)[0]
        v[at - 1] = make(1, 1, D, 6, 3e3)[0]
        run(dev, q, k, v, g, o, o, causal, 0.0000625)


def test_a_query_alone_is_the_same_with_and_without_the_mask(dev):
    """Lists of one query: the mask hides nothing, so both calls give the same bits."""
    nq, nk, H, D = [1] * 5, [2, 64, 65, 300, 9], 2, 128
    qo, ko = offsets_of(nq), offsets_of(nk)
    q, k = make(qo[-1], H, D, 1, 37.6), make(ko[-1], H, D, 2, 37.6)
    v, g = make(ko[-1], H, D, 3, 18.0), make(qo[-1], H, D, 4, 5e3)
    masked = run(dev, q, k, v, g, qo, ko, True, 0.000125)
    for x, y in zip(masked, run(dev, q, k, v, g, qo, ko, False, 0.000125)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("causal", [True, False])
def test_infinite_gradients_stay_so(dev, causal):
    """An overflow of the caller's (an infinity among the incoming gradients) reaches the
    gradients of what its query sees, as loss scaling expects it."""
    n, D, at = 130, 64, 40
    o = torch.tensor([0, n], device=dev)
    leaves = [make(n, 1, D, i, 1.0).to(dev).requires_grad_() for i in range(3)]
    g = make(n, 1, D, 4, 1.0).to(dev)
    g[at, 0, 3] = float("inf")
    dq, dk, dv = torch.autograd.grad(OPS.jagged_attention(*leaves, o, o, causal), leaves, g)
    assert not torch.isfinite(dq[at]).all() and not torch.isfinite(dk[: at + 1]).any(dim=-1).any()
    assert not torch.isfinite(dv[: at + 1, 0, 3]).any()
    others = [i for i in range(n) if i != at]
    assert torch.isfinite(dq[others]).all()
    if causal:
        assert torch.isfinite(dk[at + 1:]).all() and torch.isfinite(dv[at + 1:]).all()

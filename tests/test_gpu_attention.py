"""Attention over packed sequences on the GPU against its float64 definition
(attention_helpers; the tolerances are bounds of the roundings the kernels
make), and its refusals."""

import numpy as np
import pytest
import torch

from attention_helpers import attention, check

pytestmark = pytest.mark.gpu

DT = {"float16": torch.float16, "bfloat16": torch.bfloat16}


def offsets_of(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)


def make(rows, heads, D, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((rows, heads, D), generator=g) * scale).to(DT[dtype])


def run(dev, q, k, v, qo, ko, causal, scale, dtype, grad=None, index=torch.int64, self_attention=False):
    """Forward (and backward) on the GPU next to the definition; checks both."""
    print(f"[case] q {tuple(q.shape)} k {tuple(k.shape)} {dtype} causal={causal} lists={len(qo) - 1}", flush=True)
    qd, kd, vd = (x.to(dev) for x in (q, k, v))
    tqo = torch.from_numpy(np.asarray(qo)).to(dev, index)
    tko = None if self_attention else torch.from_numpy(np.asarray(ko)).to(dev, index)
    out, lse = torch.ops.mx_fbgemm.jagged_attention_forward(qd, kd, vd, tqo, tko, causal, scale)
    s = scale if scale is not None else 1.0 / np.sqrt(q.size(2))
    want = attention(q.double().numpy(), k.double().numpy(), v.double().numpy(), qo, ko, causal, s, dtype,
                     None if grad is None else grad.double().numpy())
    check(out.double().cpu().numpy(), want.out, want.out_tol, "out")
    check(lse.double().cpu().numpy(), want.lse, want.lse_tol, "lse")
    if grad is None:
        return out
    leaves = [x.detach().requires_grad_() for x in (qd, kd, vd)]
    o2 = torch.ops.mx_fbgemm.jagged_attention(*leaves, tqo, tko, causal, scale)
    assert torch.equal(o2, out)
    got = torch.autograd.grad(o2, leaves, grad.to(dev))
    for name, x, w, t in zip(("dq", "dk", "dv"), got, (want.dq, want.dk, want.dv),
                             (want.dq_tol, want.dk_tol, want.dv_tol)):
        check(x.double().cpu().numpy(), w, t, name)
    return out


MIXED = [0, 3, 1, 0, 33, 64, 65, 2, 127, 128, 129, 0]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("D", [8, 32, 40, 64, 72, 96, 104, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_self_attention(dev, dtype, D, causal):
    o = offsets_of(MIXED)
    n = int(o[-1])
    q, k, v, g = (make(n, 2, D, dtype, 10 * D + i) for i in range(4))
    run(dev, q, k, v, o, o, causal, None, dtype, g, self_attention=True)


@pytest.mark.parametrize("H,Hkv", [(1, 1), (4, 1), (6, 3), (8, 8), (16, 4)])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_grouped_heads(dev, H, Hkv, index):
    o = offsets_of([70, 0, 5, 200])
    n = int(o[-1])
    q, g = make(n, H, 64, "bfloat16", 1), make(n, H, 64, "bfloat16", 2)
    k, v = make(n, Hkv, 64, "bfloat16", 3), make(n, Hkv, 64, "bfloat16", 4)
    run(dev, q, k, v, o, o, True, 0.2, "bfloat16", g, index)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("causal", [True, False])
def test_more_or_fewer_keys_than_queries(dev, dtype, causal):
    """Histories before the queries; lists with fewer keys, whose first queries
    see nothing; lists without queries, without keys, without either."""
    nq = [5, 40, 130, 70, 0, 9, 0, 1, 300]
    nk = [9, 140, 20, 1, 8, 0, 0, 500, 290]
    qo, ko = offsets_of(nq), offsets_of(nk)
    q, g = make(int(qo[-1]), 4, 64, dtype, 1), make(int(qo[-1]), 4, 64, dtype, 2)
    k, v = make(int(ko[-1]), 2, 64, dtype, 3), make(int(ko[-1]), 2, 64, dtype, 4)
    out = run(dev, q, k, v, qo, ko, causal, None, dtype, g)
    if causal:
        assert torch.count_nonzero(out[qo[2]: qo[2] + 110]) == 0  # 130 queries, 20 keys
    assert torch.count_nonzero(out[qo[5]: qo[6]]) == 0            # no keys


@pytest.mark.parametrize("lists,length", [(1, 1), (70, 5), (500, 3), (5000, 1)])
def test_many_lists(dev, lists, length):
    """The list lookup takes one, two and three rounds of 64."""
    rng = np.random.default_rng(lists)
    n = rng.integers(0, 2 * length + 1, lists)
    n[-1] = length
    o = offsets_of(n)
    q, k, v, g = (make(int(o[-1]), 1, 32, "bfloat16", i) for i in range(4))
    run(dev, q, k, v, o, o, True, None, "bfloat16", g)


@pytest.mark.parametrize("lists,most", [(20, 1000), (70, 260), (1100, 20)])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("causal", [True, False])
def test_many_tiles(dev, lists, most, index, causal):
    """Enough tiles for an order of their own: lists of unlike lengths, rows of no
    list at both ends, and other lengths for the keys."""
    rng = np.random.default_rng(lists)
    nq, nk = rng.integers(0, most + 1, lists), rng.integers(0, most + 1, lists)
    nq[lists // 2], nk[lists // 3] = 700, 0
    qo, ko = offsets_of(nq) + 5, offsets_of(nk) + 300
    Nq, Nk = int(qo[-1]) + 600, int(ko[-1]) + 1
    q, g = make(Nq, 64, 8, "bfloat16", 1), make(Nq, 64, 8, "bfloat16", 2)
    k, v = make(Nk, 4, 8, "bfloat16", 3), make(Nk, 4, 8, "bfloat16", 4)
    run(dev, q, k, v, qo, ko, causal, None, "bfloat16", g, index)


@pytest.mark.parametrize("Hkv", [16, 32, 64])
@pytest.mark.parametrize("causal", [True, False])
def test_heads_of_a_block(dev, Hkv, causal):
    """Four, two and one query heads of a block, on tiles found by rank: more
    keys than queries, fewer, and a single query."""
    qo, ko = offsets_of([400, 1, 330, 410]), offsets_of([900, 1300, 300, 1200])
    q, g = make(int(qo[-1]), 64, 8, "bfloat16", 1), make(int(qo[-1]), 64, 8, "bfloat16", 2)
    k, v = make(int(ko[-1]), Hkv, 8, "bfloat16", 3), make(int(ko[-1]), Hkv, 8, "bfloat16", 4)
    run(dev, q, k, v, qo, ko, causal, None, "bfloat16", g)


@pytest.mark.parametrize("H,Hkv", [(8, 1), (3, 3)])
@pytest.mark.parametrize("D", [24, 64, 96, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_shared_out_queries(dev, H, Hkv, D, causal):
    """Few keys under many queries: each key's gradients are sums of several
    shares, some of them empty, some lists without queries or keys."""
    qo, ko = offsets_of([0, 1, 900, 70, 300]) + 2, offsets_of([40, 3, 500, 0, 310]) + 1
    Nq, Nk = int(qo[-1]) + 3, int(ko[-1]) + 5
    q, g = make(Nq, H, D, "float16", 1), make(Nq, H, D, "float16", 2)
    k, v = make(Nk, Hkv, D, "float16", 3), make(Nk, Hkv, D, "float16", 4)
    run(dev, q, k, v, qo, ko, causal, None, "float16", g)


@pytest.mark.parametrize("dtype,D", [("float16", 128), ("bfloat16", 128), ("bfloat16", 64)])
def test_long_lists(dev, dtype, D):
    o = offsets_of([1500, 777])
    n = int(o[-1])
    q, g = make(n, 2, D, dtype, 1), make(n, 2, D, dtype, 2)
    k, v = make(n, 1, D, dtype, 3), make(n, 1, D, dtype, 4)
    run(dev, q, k, v, o, o, True, None, dtype, g)


def test_large_scores(dev):
    """Scores of +-60: probabilities of one key dominate, maxima grow along the list."""
    o = offsets_of([400])
    q, k, v, g = (make(400, 2, 64, "float16", i, 3.0 if i < 2 else 1.0) for i in range(4))
    run(dev, q, k, v, o, o, True, None, "float16", g)


def test_rows_of_no_list(dev):
    """Rows before the first and after the last offset: zeros, and no part in the rest."""
    o = np.array([40, 100, 150], np.int64)
    q, k, v, g = (make(300, 2, 64, "bfloat16", i) for i in range(4))
    for x in (k, v):
        x[:40] = float("nan")
        x[150:] = float("inf")
    out = run(dev, q, k.where(torch.isfinite(k), torch.zeros(())), v.where(torch.isfinite(v), torch.zeros(())),
              o, o, True, None, "bfloat16", g)
    to = torch.from_numpy(o).to(dev)
    again = torch.ops.mx_fbgemm.jagged_attention(q.to(dev), k.to(dev), v.to(dev), to, to, True)
    assert torch.equal(out, again)
    assert torch.count_nonzero(out[:40]) == 0 and torch.count_nonzero(out[150:]) == 0


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_other_lists_do_not_reach_in(dev, bad):
    """A list next to one full of NaN or infinities gives what it gives alone."""
    n = [37, 50, 91]
    o = torch.from_numpy(offsets_of(n)).to(dev)
    q, k, v, g = (make(sum(n), 2, 64, "bfloat16", i).to(dev) for i in range(4))
    for x in (q, k, v, g):
        x[37:87] = bad
    def both(s, off):
        leaves = [x[s].detach().clone().requires_grad_() for x in (q, k, v)]
        out = torch.ops.mx_fbgemm.jagged_attention(*leaves, off, off, True)
        return out, torch.autograd.grad(out, leaves, g[s])
    out, grads = both(slice(None), o)
    for s in (slice(0, 37), slice(87, 178)):
        m = s.stop - s.start
        alone, gal = both(s, torch.tensor([0, m], device=dev))
        assert torch.equal(out[s], alone)
        for x, y in zip(grads, gal):
            assert torch.equal(x[s], y)


def test_strides(dev):
    """Views of a fused projection, heads before rows, shared heads and rows that
    have to be copied (odd strides, unaligned starts) give the contiguous result."""
    o = torch.from_numpy(offsets_of([60, 0, 140])).to(dev)
    n, H, D = 200, 4, 64
    q, k, v, g = (make(n, H, D, "bfloat16", i).to(dev) for i in range(4))

    def both(q, k, v, g):
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        out = torch.ops.mx_fbgemm.jagged_attention(*leaves, o, o, True)
        return (out, *torch.autograd.grad(out, leaves, g))

    want = both(q, k, v, g)

    def same(*args):
        for x, y in zip(both(*args), want):
            assert torch.equal(x, y)

    fused = torch.cat([q, k, v], 1)
    same(fused[:, :H], fused[:, H:2 * H], fused[:, 2 * H:], g)
    same(*(x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v, g)))
    wide = torch.zeros((n, H, D + 1), dtype=q.dtype, device=dev)
    wide[:, :, :D] = q
    same(wide[:, :, :D], k, v, g)
    flat = torch.zeros(n * H * D + 1, dtype=q.dtype, device=dev)
    flat[1:] = k.reshape(-1)
    same(q, flat[1:].view(n, H, D), v, g)
    last = q.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    same(last, k, v, g)
    # An expanded key-value head, and an expanded gradient.
    one = k[:, :1].expand(n, H, D)
    ones = torch.ones((), dtype=q.dtype, device=dev).expand(n, H, D)
    a = both(q, one, v, ones)
    b = both(q, one.contiguous(), v, ones.contiguous())
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_same_bits_every_time_and_other_streams(dev):
    o = torch.from_numpy(offsets_of([300, 20, 411])).to(dev)
    q, g = (make(731, 8, 64, "bfloat16", i).to(dev) for i in (0, 1))
    k, v = (make(731, 2, 64, "bfloat16", i).to(dev) for i in (2, 3))

    def both():
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        out = torch.ops.mx_fbgemm.jagged_attention(*leaves, o, o, True)
        return (out, *torch.autograd.grad(out, leaves, g))

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
    torch.cuda.current_stream().wait_stream(side)
    for got in (both(), other):
        for x, y in zip(got, want):
            assert torch.equal(x, y)


def test_only_the_gradients_asked_for(dev):
    o = torch.tensor([0, 50], device=dev)
    q, k, v, g = (make(50, 2, 32, "float16", i).to(dev) for i in range(4))
    all3 = torch.autograd.grad(torch.ops.mx_fbgemm.jagged_attention(
        *(x.requires_grad_() for x in (q, k, v)), o), (q, k, v), g)
    for i in range(3):
        leaves = [x.detach() for x in (q, k, v)]
        leaves[i].requires_grad_()
        out = torch.ops.mx_fbgemm.jagged_attention(*leaves, o)
        assert torch.equal(torch.autograd.grad(out, leaves[i], g)[0], all3[i])
    with torch.no_grad():
        assert not torch.ops.mx_fbgemm.jagged_attention(q, k, v, o).requires_grad


def test_gradient_against_differences(dev):
    """The gradients' slope along a direction against a difference of the float64 loss."""
    n, H, D = 90, 2, 32
    o = offsets_of([50, 40])
    q, k, v, g = (make(n, H, D, "float16", 20 + i) for i in range(4))
    leaves = [x.to(dev).requires_grad_() for x in (q, k, v)]
    to = torch.from_numpy(o).to(dev)
    out = torch.ops.mx_fbgemm.jagged_attention(*leaves, to, to, True, 0.2)
    grads = torch.autograd.grad(out, leaves, g.to(dev))
    x = [t.double().numpy() for t in (q, k, v)]
    r = attention(*x, o, o, True, 0.2, "float16", g.double().numpy())
    rng = np.random.default_rng(5)
    for i, (got, tol) in enumerate(zip(grads, (r.dq_tol, r.dk_tol, r.dv_tol))):
        step = rng.choice([-1.0, 1.0], got.shape)
        def loss(t):
            y = list(x)
            y[i] = y[i] + t * step
            return float((attention(*y, o, o, True, 0.2, "float16").out * g.double().numpy()).sum())
        diff = (loss(1e-5) - loss(-1e-5)) / 2e-5
        # The elements' bounds add up at most.
        assert abs(float((got.double().cpu().numpy() * step).sum()) - diff) <= tol.sum() + 1e-6 * abs(diff)


def test_empty(dev):
    op = torch.ops.mx_fbgemm.jagged_attention
    z = torch.zeros((0, 2, 32), dtype=torch.float16, device=dev, requires_grad=True)
    o = torch.tensor([0], device=dev)
    out = op(z, z, z, o)
    assert out.shape == (0, 2, 32)
    assert torch.autograd.grad(out, z, torch.zeros_like(z))[0].shape == z.shape
    q = make(5, 2, 32, "float16", 0).to(dev).requires_grad_()
    o = torch.tensor([0, 5], device=dev)
    none = torch.tensor([0, 0], device=dev)
    out = op(q, z, z, o, none)
    assert torch.count_nonzero(out) == 0
    assert torch.count_nonzero(torch.autograd.grad(out, q, torch.ones_like(q))[0]) == 0
    kv = make(5, 2, 32, "float16", 1).to(dev).requires_grad_()
    out = op(z, kv, kv, none, o)
    assert torch.count_nonzero(torch.autograd.grad(out, kv, torch.zeros_like(z))[0]) == 0


def test_refusals(dev):
    op = torch.ops.mx_fbgemm.jagged_attention
    x = torch.zeros((4, 2, 32), dtype=torch.float16, device=dev)
    o = torch.tensor([0, 4], device=dev)
    for args in [(x.float(), x.float(), x.float(), o),                  # fp32
                 (x, x.bfloat16(), x, o),                               # mixed types
                 (x, x, x, o.cpu()), (x.cpu(), x, x, o),                # devices
                 (x, x, x, o.float()), (x, x, x, o.view(1, 2)),         # offsets
                 (x, x, x, o, o.int()), (x, x, x, o, torch.tensor([0, 2, 4], device=dev)),
                 (x[:, :, :20], x[:, :, :20], x[:, :, :20], o),         # width no multiple of 8
                 (*(torch.zeros((4, 2, 136), dtype=torch.float16, device=dev),) * 3, o),
                 (x, x[:, :, :16], x[:, :, :16], o), (x, x[:3], x, o),
                 (x[:, :1], x, x, o),                                   # heads
                 (x, x[:2], x[:2], o),                                  # rows without k_offsets
                 (x.view(4, 64), x, x, o),
                 (x, x, x, o, o, True, 0.0), (x, x, x, o, o, True, -1.0),
                 (x, x, x, o, o, True, float("nan"))]:
        with pytest.raises((RuntimeError, NotImplementedError)):
            op(*args)
    q = x.detach().requires_grad_()
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(op(q, x, x, o).sum(), q, create_graph=True)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("H,D,n", [(1, 64, 200), (4, 128, 1100)])
def test_masked_keys_and_values_do_not_show(dev, bad, H, D, n):
    """Under the causal mask what later events hold reaches no earlier one, and
    what a query sees of it reaches the query."""
    o = torch.tensor([0, n], device=dev)
    q, k, v = (make(n, H, D, "bfloat16", i).to(dev) for i in range(3))
    want = torch.ops.mx_fbgemm.jagged_attention(q, k, v, o)
    for at in (1, 70, n - 1):
        for which in (k, v):
            keep = which[at].clone()
            which[at] = bad
            got = torch.ops.mx_fbgemm.jagged_attention(q, k, v, o)
            which[at] = keep
            # Rows that share a wave with a bad one are worked out another way:
            # equal to the two ways' roundings.
            g, w = got[:at].double(), want[:at].double()
            assert torch.isfinite(g).all()
            assert ((g - w).norm() <= 2 * 2.0 ** -8 * w.norm())
            assert torch.equal(got[: at // 128 * 128], want[: at // 128 * 128])
            if which is v:
                assert not torch.isfinite(got[at:]).any()
            else:
                assert not torch.isfinite(got[at:]).all()


@pytest.mark.parametrize("low", [-60000.0, -3.0e38])
def test_scores_of_the_types_lowest_values(dev, low):
    """Keys that give scores near the lowest numbers: weights of zero, no NaN."""
    dtype = "float16" if low > -65505 else "bfloat16"
    n = 130
    q, k, v = (make(n, 1, 32, dtype, i) for i in range(3))
    q = q.abs()
    k[10:20] = low
    o = offsets_of([n])
    to = torch.from_numpy(o).to(dev)
    out = torch.ops.mx_fbgemm.jagged_attention(q.to(dev), k.to(dev), v.to(dev), to, to, True)
    assert torch.isfinite(out).all()
    keep = [i for i in range(n) if not 10 <= i < 20]
    some = torch.ops.mx_fbgemm.jagged_attention(
        q[keep].to(dev), k[keep].to(dev), v[keep].to(dev), torch.tensor([0, 120], device=dev),
        torch.tensor([0, 120], device=dev), True)
    g, w = out[keep].double(), some.double()
    assert ((g - w).norm() <= 2 * 2.0 ** -8 * w.norm())


@pytest.mark.parametrize("H,Hkv,D,n", [(1, 1, 64, 200), (4, 2, 128, 1100)])
def test_masked_pairs_do_not_show_in_gradients(dev, H, Hkv, D, n):
    """What a row holds reaches only gradients of pairs that the mask lets through:
    a bad key or value not the earlier queries', a bad query or incoming gradient
    not the later keys'."""
    o = torch.tensor([0, n], device=dev)
    q, g = (make(n, H, D, "bfloat16", i) for i in (0, 1))
    k, v = (make(n, Hkv, D, "bfloat16", i) for i in (2, 3))
    r = attention(*(x.double().numpy() for x in (q, k, v)), [0, n], [0, n], True, D ** -0.5, "bfloat16",
                  g.double().numpy())
    q, k, v, g = (x.to(dev) for x in (q, k, v, g))

    def near(got, want, tol, s, what):
        check(got[s].double().cpu().numpy(), want[s], tol[s], what)

    for at in (1, 70, n - 2):
        for name, x in (("q", q), ("k", k), ("v", v), ("g", g)):
            keep = x[at].clone()
            x[at] = float("nan")
            leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
            out = torch.ops.mx_fbgemm.jagged_attention(*leaves, o)
            dq, dk, dv = torch.autograd.grad(out, leaves, g)
            x[at] = keep
            if name in "kv":
                near(dq, r.dq, r.dq_tol, slice(0, at), f"dq before a bad {name}")
                assert torch.isnan(dq[at:]).all()
            else:
                near(dk, r.dk, r.dk_tol, slice(at + 1, n), f"dk after a bad {name}")
                near(dv, r.dv, r.dv_tol, slice(at + 1, n), f"dv after a bad {name}")
                near(dq, r.dq, r.dq_tol, slice(at + 1, n), f"dq after a bad {name}")
                assert torch.isnan(dk[: at + 1]).all()

"""Rotation by position on the GPU: bit for bit against the formulas with every
operation rounded to fp32, its gradient, and its refusals."""

import numpy as np
import pytest
import torch

from mx_fbgemm.sequence_attention import rotary_table
from rows_helpers import DT, angles, make, rotate

pytestmark = pytest.mark.gpu

OPS = torch.ops.mx_fbgemm


def same(got, want, what=""):
    """Equal bits; every NaN is alike."""
    got, want = got.detach().cpu(), want.to(got.dtype)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), what
    a, b = got.masked_fill(nan, 0).view(torch.int16), want.masked_fill(nan, 0).view(torch.int16)
    assert torch.equal(a, b), (what, int((a != b).sum()))


def lists(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(int).tolist()


def run(dev, lengths, H, D, R, dtype, interleaved=False, starts=None, index=torch.int64, positions=None, x=None,
        extra=0):
    off = lists(lengths)
    print(f"[case] {len(lengths)} lists, {off[-1]} rows, H={H} D={D} R={R} {dtype} {interleaved}", flush=True)
    if x is None:
        x = make((off[-1] + extra, H, D), dtype, 1)
    most = max([n + (starts[b] if starts else 0) for b, n in enumerate(lengths)] + [1])
    table = angles(positions if positions is not None else most, R)
    s = torch.tensor(starts, dtype=index, device=dev) if starts else None
    y = OPS.jagged_rotary(x.to(dev), torch.tensor(off, dtype=index, device=dev), table.to(dev), s, interleaved)
    want = rotate(x, off, table, starts, interleaved)
    same(y, want)
    return x, y, table, off


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,R", [(8, 8), (16, 8), (24, 24), (32, 32), (40, 40), (40, 16), (64, 64), (64, 24), (72, 72),
                                 (96, 96), (104, 56), (128, 128), (128, 64), (128, 8)])
def test_widths(dev, dtype, interleaved, D, R):
    run(dev, [3, 0, 70, 1], 3, D, R, dtype, interleaved, starts=[5, 0, 0, 9])


@pytest.mark.parametrize("H", [1, 2, 5, 17, 64, 130])
def test_heads(dev, H):
    run(dev, [9, 1, 0, 4], H, 64, 64, "bfloat16")


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("B,most", [(1, 1), (1, 5000), (300, 3), (2000, 1), (70, 200)])
def test_lists(dev, index, B, most):
    rng = np.random.default_rng(B + most)
    n = [int(v) for v in rng.integers(0, most + 1, B)]
    n[0] = most
    run(dev, n, 2, 32, 32, "float16", starts=[int(v) for v in rng.integers(0, 50, B)], index=index)


@pytest.mark.parametrize("H,D", [(1, 8), (2, 64), (20, 128)])
def test_many_empty_lists_between_rows(dev, H, D):
    n = [1] + [0] * 700 + [2] + [0] * 64 + [1] + [0] * 63 + [40] + [0] * 130
    run(dev, n, H, D, D, "bfloat16")


def test_far_positions(dev):
    """Angles come from the table, which is rounded from 64 bits: near 2^20 the
    rotation keeps its accuracy (fp16: one rounding, plus the table's and the
    products' 2^-24 each)."""
    P, R = 1 << 20, 64
    table = rotary_table(P, R, device=dev)
    x = make((64, 2, R), "float16", 3)
    start = P - 64
    y = OPS.jagged_rotary(x.to(dev), torch.tensor([0, 64], device=dev), table, torch.tensor([start], device=dev))
    w = 10000.0 ** (-2 * np.arange(R // 2) / R)
    a = (start + np.arange(64))[:, None] * w
    z = (x[..., :R // 2].double().numpy() + 1j * x[..., R // 2:].double().numpy()) * np.exp(1j * a)[:, None]
    want = np.concatenate([z.real, z.imag], -1)
    size = np.abs(np.concatenate([z, z], -1))
    off = np.abs(y.double().cpu().numpy() - want)
    # The angle itself, in 64 bits on both sides, is off by up to 2^20 2^-53.
    assert (off <= 2.0 ** -11 * np.abs(want) + size * (6 * 2.0 ** -24 + 2.0 ** -32) + 2.0 ** -25).all()


def test_rows_of_no_list_and_positions_without_angles(dev):
    x = make((10, 2, 32), "bfloat16", 1)
    table = angles(4, 16)
    off, starts = [2, 4, 4, 8], [1, 0, 2]
    y = OPS.jagged_rotary(x.to(dev), torch.tensor(off, device=dev), table.to(dev), torch.tensor(starts, device=dev))
    want = rotate(x, off, table, starts)
    same(y, want)
    assert torch.count_nonzero(y[:2]) == 0 and torch.count_nonzero(y[8:]) == 0
    assert torch.isnan(y[6:8, :, :16]).all() and torch.equal(y[4:8, :, 16:].cpu(), x[4:8, :, 16:])
    y = OPS.jagged_rotary(x.to(dev), torch.tensor(off, device=dev), table.to(dev),
                          torch.tensor([-1, 0, 2 ** 40], device=dev))
    assert torch.isnan(y[2:8, :, :16]).all() and torch.count_nonzero(y[:2]) == 0
    y = OPS.jagged_rotary(x.to(dev), torch.tensor(off, device=dev), table[:0].to(dev))
    assert torch.isnan(y[2:8, :, :16]).all()


def test_views(dev):
    """Queries and keys in one projection's output; a transposed, an offset and a
    stretched view; a table cut out of a longer one."""
    off = torch.tensor([0, 5, 9], device=dev)
    table = angles(9, 48).to(dev)
    x = make((9, 12, 64), "float16", 1).to(dev)
    want = OPS.jagged_rotary(x[:, :8].contiguous(), off, table)
    for v in (x[:, :8], x[:, :8].transpose(0, 1).contiguous().transpose(0, 1),
              torch.cat([x[:, :8], x[:, :8]], 2)[:, :, 64:],
              torch.cat([x[:, :8, :1], x[:, :8]], 2)[:, :, 1:]):  # (the last is copied: rows at odd addresses)
        assert torch.equal(OPS.jagged_rotary(v, off, table), want)
    one = x[:, :1].contiguous()
    assert torch.equal(OPS.jagged_rotary(one.expand(9, 8, 64), off, table),
                       OPS.jagged_rotary(one.repeat(1, 8, 1), off, table))
    wide = torch.cat([table, table], 1)
    assert torch.equal(OPS.jagged_rotary(x[:, :8], off, wide[:, :24]), want)
    assert torch.equal(OPS.jagged_rotary(x[:, :8], off.int(), table, torch.zeros(2, dtype=torch.int64, device=dev)), want)


def test_infinities_and_nan_stay_in_their_pairs(dev):
    x = make((4, 1, 32), "bfloat16", 1)
    x[1, 0, 3], x[2, 0, 20] = float("inf"), float("nan")
    table = angles(4, 32)
    y = OPS.jagged_rotary(x.to(dev), torch.tensor([0, 4], device=dev), table.to(dev))
    same(y, rotate(x, [0, 4], table))
    fine = torch.isfinite(y.cpu())
    assert int((~fine).sum()) == 4 and not fine[1, 0, 3] and not fine[1, 0, 19] and not fine[2, 0, 4] and not fine[2, 0, 20]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_gradient(dev, dtype, interleaved):
    """The rotation back, bit for bit; and, as the operator is linear, the inner
    product <y(dx), g> = <dx, x_grad(g)> of values rounded once each."""
    off, starts = [0, 7, 7, 40], [3, 0, 100]
    x = make((43, 3, 96), dtype, 1).to(dev).requires_grad_()
    g = make((43, 3, 96), dtype, 2)
    table = angles(200, 80)
    o, s, t = torch.tensor(off, device=dev), torch.tensor(starts, device=dev), table.to(dev)
    y = OPS.jagged_rotary(x, o, t, s, interleaved)
    dx, = torch.autograd.grad(y, x, g.to(dev))
    same(dx, rotate(g, off, table, starts, interleaved, sign=-1))
    same(OPS.jagged_rotary_backward(g.to(dev), o, t, s, interleaved), dx.cpu())
    d = make((43, 3, 96), dtype, 3)
    yd = OPS.jagged_rotary(d.to(dev), o, t, s, interleaved).double().cpu()
    left, right = (yd * g.double()).sum(), (d.double() * dx.double().cpu()).sum()
    u = 2.0 ** -11 if dtype == "float16" else 2.0 ** -8
    assert abs(left - right) <= (u + 2.0 ** -20) * ((yd * g.double()).abs().sum() + (d.double() * dx.double().cpu()).abs().sum()) + 1e-4


def test_gradient_of_strided_and_expanded_gradients(dev):
    off = torch.tensor([0, 5], device=dev)
    table = angles(5, 32).to(dev)
    x = make((5, 4, 32), "float16", 1).to(dev).requires_grad_()
    y = OPS.jagged_rotary(x, off, table)
    y.sum().backward()  # an expanded gradient, of strides 0
    want = OPS.jagged_rotary_backward(torch.ones_like(x), off, table)
    assert torch.equal(x.grad, want)


def test_second_derivative_and_no_gradient_of_the_table(dev):
    off = torch.tensor([0, 5], device=dev)
    table = angles(5, 32).to(dev)
    x = make((5, 2, 32), "bfloat16", 1).to(dev).requires_grad_()
    g = make((5, 2, 32), "bfloat16", 2).to(dev).requires_grad_()
    y = OPS.jagged_rotary(x, off, table)
    dx, = torch.autograd.grad(y, x, g, create_graph=True)
    w = make((5, 2, 32), "bfloat16", 3).to(dev)
    dg, = torch.autograd.grad(dx, g, w)
    assert torch.equal(dg, OPS.jagged_rotary(w, off, table))
    with pytest.raises(RuntimeError, match="gradient of its table"):
        OPS.jagged_rotary(x, off, table.clone().requires_grad_())
    with pytest.raises(NotImplementedError), torch.autograd.forward_ad.dual_level():
        OPS.jagged_rotary(torch.autograd.forward_ad.make_dual(x.detach(), g.detach()), off, table)


def test_other_stream_and_graph(dev):
    off = torch.tensor([0, 30, 50], device=dev)
    table = angles(30, 64).to(dev)
    x = make((50, 4, 64), "bfloat16", 1).to(dev)
    want = OPS.jagged_rotary(x, off, table)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = OPS.jagged_rotary(x, off, table)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    leaf = x.clone().requires_grad_()
    grad = make((50, 4, 64), "bfloat16", 2).to(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = OPS.jagged_rotary(leaf, off, table)
        dx, = torch.autograd.grad(y, leaf, grad)
    for seed in (5, 6, 7):
        with torch.no_grad():
            leaf.copy_(make((50, 4, 64), "bfloat16", seed))
        off.copy_(torch.tensor([0, 5 * seed - 5, 50]))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, OPS.jagged_rotary(leaf.detach(), off, table))
        assert torch.equal(dx, OPS.jagged_rotary_backward(grad, off, table))


def test_empty(dev):
    table = angles(4, 32).to(dev)
    for shape in ((0, 2, 32), (3, 0, 32)):
        x = torch.zeros(shape, dtype=torch.float16, device=dev)
        assert OPS.jagged_rotary(x, torch.tensor([0, shape[0]], device=dev), table).shape == shape
    x = make((3, 2, 32), "float16", 1).to(dev)
    none = torch.tensor([0], device=dev)
    assert torch.count_nonzero(OPS.jagged_rotary(x, none, table)) == 0
    assert torch.count_nonzero(OPS.jagged_rotary(x, none, table, none[:0])) == 0


def test_refusals(dev):
    x = torch.zeros((4, 2, 32), dtype=torch.float16, device=dev)
    off, table, starts = torch.tensor([0, 1, 4], device=dev), angles(4, 32).to(dev), torch.zeros(2, dtype=torch.int64, device=dev)
    for args in [(x.float(), off, table), (x[:, :, :12], off, table), (x[0], off, table), (x, off.float(), table),
                 (x, off.view(1, 3), table), (x, off[:0], table), (x, off, table.double()), (x, off, table.half()),
                 (x, off, table[0]), (x, off, table[:, :, :1]), (x, off, table[:, :3]), (x, off, table[:, :0]),
                 (x[:, :, :16], off, table), (x, off.cpu(), table), (x, off, table.cpu()),
                 (x, off, table, starts[:1]), (x, off, table, starts.float()), (x, off, table, starts.cpu()),
                 (torch.zeros((4, 2, 136), dtype=torch.float16, device=dev), off, table), (x.cpu(), off, table)]:
        with pytest.raises((RuntimeError, NotImplementedError)):
            OPS.jagged_rotary(*args)

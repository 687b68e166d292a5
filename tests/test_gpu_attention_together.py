"""The attention operators as they are used together: the sequence example, the
cache object, captured graphs, and the C-ABI through ctypes."""

import ctypes
import importlib.util
from pathlib import Path

import numpy as np
import pytest
import torch

from attention_helpers import attention, check, paged_attention
from mx_fbgemm.sequence_attention import PagedSequenceCache

pytestmark = pytest.mark.gpu

REPO = Path(__file__).resolve().parents[1]
LIB = REPO / "torchlib-xpu_amd" / "mx_fbgemm" / "lib" / "libmx_fbgemm_kernels.so"
OPS = torch.ops.mx_fbgemm


def make(shape, seed, dtype=torch.bfloat16):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def test_the_example_trains_and_serves(dev):
    spec = importlib.util.spec_from_file_location("sequence_model", REPO / "examples" / "sequence_model.py")
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    torch.manual_seed(0)
    model = m.SequenceModel(200)
    before = model.table.weights_dev.clone()
    losses = m.train(model, 16, 60, 200, 8)
    assert losses[-1] < losses[0] and not torch.equal(before, model.table.weights_dev)
    got, want = m.serve(model, 16, 60, 200, 3)
    # Each side rounds its probabilities and its result to bf16.
    assert (got - want).float().norm() <= 2 * 2.0 ** -8 * want.float().norm()


def test_cache_object(dev):
    """Histories of other lengths, events one by one, a sequence that leaves and
    one that takes its pages, calls on some of the sequences in any order."""
    H, Hkv, D = 4, 2, 32
    c = PagedSequenceCache(pages=16, page_size=8, heads=Hkv, head_dim=D, max_sequences=3, max_length=64)
    held = {}

    def append(names, counts, seed):
        n = sum(counts)
        k, v = make((n, Hkv, D), seed), make((n, Hkv, D), seed + 1)
        c.append(names, counts, k.to(dev), v.to(dev))
        at = 0
        for s, m in zip(names, counts):
            ok, ov = held.get(s, (k[:0], v[:0]))
            held[s] = (torch.cat([ok, k[at:at + m]]), torch.cat([ov, v[at:at + m]]))
            at += m

    def attend(names, seed):
        q = make((len(names), H, D), seed)
        out = c.attend(names, q.to(dev))
        want, tol = paged_attention(q.double().numpy(), [held[s][0].double().numpy() for s in names],
                                    [held[s][1].double().numpy() for s in names], D ** -0.5, "bfloat16")
        check(out.double().cpu().numpy(), want, tol, "out")

    a, b = c.add(), c.add()
    append([a, b], [20, 3], 10)
    attend([a, b], 20)
    append([b], [1], 30)
    attend([b, a], 21)
    c.remove(a)
    del held[a]
    x, y = c.add(), c.add()
    append([y, x, b], [40, 0, 9], 40)
    attend([y, b, x], 22)
    assert c.length(b) == 13 and c.length(x) == 0
    with pytest.raises(RuntimeError, match="pages needed"):
        append([x, y, b], [60, 8, 40], 50)
    attend([b], 23)


def test_graph_replays_match_eager(dev):
    """One training step and one serving step captured; new inputs before every
    replay, eager work and a synchronisation between them."""
    n, H, Hkv, D, B = 300, 4, 2, 64, 3
    o = torch.tensor([0, 100, 130, 300], device=dev)
    q, g = (torch.empty((n, H, D), dtype=torch.bfloat16, device=dev) for _ in range(2))
    k, v = (torch.empty((n, Hkv, D), dtype=torch.bfloat16, device=dev) for _ in range(2))
    kc, vc = (torch.zeros((12, 16, Hkv, D), dtype=torch.bfloat16, device=dev) for _ in range(2))
    table = torch.arange(12, dtype=torch.int32, device=dev).view(B, 4)
    starts, lengths = torch.zeros(B, dtype=torch.int32, device=dev), torch.ones(B, dtype=torch.int32, device=dev)
    one = torch.arange(B + 1, device=dev)

    def step():
        out, lse = OPS.jagged_attention_forward(q, k, v, o)
        grads = OPS.jagged_attention_backward(g, q, k, v, out, lse, o)
        OPS.paged_cache_append(k[:B], v[:B], one, starts, kc, vc, table)
        return (out, *grads, OPS.paged_cache_attention(q[:B], kc, vc, table, lengths))

    def fill(i):
        for j, t in enumerate((q, k, v, g)):
            t.copy_(make(t.shape, 10 * i + j))
        starts.fill_(i)
        lengths.fill_(i + 1)

    fill(0)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    kc.zero_(), vc.zero_()
    for i in range(4):
        fill(i)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in held]
        want = step()  # the same rows to the same slots
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)


class Tensor3(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("row_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64)]


class Problem(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int32), ("index_bytes", ctypes.c_int32), ("q_offsets", ctypes.c_void_p),
                ("k_offsets", ctypes.c_void_p), ("B", ctypes.c_int64), ("Nq", ctypes.c_int64),
                ("Nk", ctypes.c_int64), ("H", ctypes.c_int32), ("Hkv", ctypes.c_int32), ("D", ctypes.c_int32),
                ("causal", ctypes.c_int32), ("scale", ctypes.c_float)]


def test_forward_through_ctypes(dev):
    lib = ctypes.CDLL(str(LIB))
    lib.mx_last_error.restype = ctypes.c_char_p
    P = ctypes.c_void_p
    T3 = ctypes.POINTER(Tensor3)
    lib.mx_jagged_attention_forward.argtypes = [ctypes.POINTER(Problem), T3, T3, T3, P, P, P,
                                                ctypes.c_size_t, P]
    n, H, Hkv, D = 50, 4, 2, 32
    q, k, v = make((n, H, D), 1), make((n, Hkv, D), 2), make((n, Hkv, D), 3)
    o = np.array([0, 20, 50])
    qd, kd, vd, od = q.to(dev), k.to(dev), v.to(dev), torch.from_numpy(o).to(dev)
    out, lse = torch.empty_like(qd), torch.empty((H, n), device=dev)
    p = Problem(2, 8, od.data_ptr(), od.data_ptr(), 2, n, n, H, Hkv, D, 1, 0.25)
    args = [Tensor3(x.data_ptr(), x.stride(0), x.stride(1)) for x in (qd, kd, vd)]
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.mx_jagged_attention_forward(p, *args, out.data_ptr(), lse.data_ptr(), None, 0, stream) == 0
    r = attention(*(x.double().numpy() for x in (q, k, v)), o, o, True, 0.25, "bfloat16")
    check(out.double().cpu().numpy(), r.out, r.out_tol, "out")
    check(lse.double().cpu().numpy(), r.lse, r.lse_tol, "lse")
    # Refused before any launch, with a message.
    for field, bad in (("dtype", 0), ("index_bytes", 2), ("H", 5), ("D", 12), ("D", 136), ("scale", 0.0),
                       ("B", -1), ("Nq", 2 ** 31)):
        keep = getattr(p, field)
        setattr(p, field, bad)
        assert lib.mx_jagged_attention_forward(p, *args, out.data_ptr(), lse.data_ptr(), None, 0, stream) == -1
        assert lib.mx_last_error()
        setattr(p, field, keep)
    for bad in (Tensor3(qd.data_ptr() + 2, H * D, D), Tensor3(qd.data_ptr(), D - 8, D),
                Tensor3(qd.data_ptr(), H * D + 4, D), Tensor3(qd.data_ptr(), 2 ** 24, D), Tensor3(0, H * D, D)):
        assert lib.mx_jagged_attention_forward(p, bad, args[1], args[2], out.data_ptr(), None, None, 0, stream) == -1
    lib.mx_jagged_attention_backward_workspace_bytes.restype = ctypes.c_size_t
    lib.mx_jagged_attention_backward_workspace_bytes.argtypes = [ctypes.POINTER(Problem)]
    assert lib.mx_jagged_attention_backward_workspace_bytes(p) == n * H * 8
    lib.mx_jagged_attention_backward.argtypes = [ctypes.POINTER(Problem), T3, T3, T3, T3, T3, P, P, P, P, P,
                                                 ctypes.c_size_t, P]
    o3 = Tensor3(out.data_ptr(), H * D, D)
    assert lib.mx_jagged_attention_backward(p, *args, o3, o3, lse.data_ptr(), out.data_ptr(), None, None, None,
                                            0, stream) == -4

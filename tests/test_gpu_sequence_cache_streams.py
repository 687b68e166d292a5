"""PagedSequenceCache's calls only enqueue work: none waits for the stream, whatever it
has to tell the device."""

import pytest
import torch

from attention_helpers import check, paged_attention
from mx_fbgemm.sequence_attention import PagedSequenceCache

pytestmark = pytest.mark.gpu

H, Hkv, D = 4, 2, 32


def make(shape, seed, dev):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).bfloat16().to(dev)


def cache():
    return PagedSequenceCache(pages=64, page_size=4, heads=Hkv, head_dim=D, max_sequences=8, max_length=64)


def calls(c, rows):
    """Prompts, single events that need pages and that do not, names in an order of
    their own, and a sequence that leaves; outputs and what each should see."""
    a, b, d = (c.add() for _ in range(3))
    seen = {s: [] for s in (a, b, d)}
    outs = []

    def append(names, counts):
        n = sum(counts)
        k, v = rows[0][:n], rows[1][:n]
        c.append(names, counts, k, v)
        at = 0
        for s, m in zip(names, counts):
            seen[s].append((at, m))
            at += m

    def attend(names):
        outs.append((list(names), {s: list(seen[s]) for s in names}, c.attend(names, rows[2][: len(names)])))

    append([a, b, d], [7, 1, 4])
    attend([a, b, d])
    for _ in range(5):
        append([d, a], [1, 1])
        attend([a, d])
    c.remove(a)
    append([b], [9])
    attend([d, b])
    return outs


def compare(outs, rows):
    k, v, q = (x.double().cpu().numpy() for x in rows)
    for names, seen, out in outs:
        keys = [k[[i for at, m in seen[s] for i in range(at, at + m)]] for s in names]
        values = [v[[i for at, m in seen[s] for i in range(at, at + m)]] for s in names]
        want, tol = paged_attention(q[: len(names)], keys, values, D ** -0.5, "bfloat16")
        check(out.double().cpu().numpy(), want, tol, "out")


def inputs(dev):
    return make((12, Hkv, D), 1, dev), make((12, Hkv, D), 2, dev), make((3, H, D), 3, dev)


def test_no_call_synchronizes(dev):
    rows, c = inputs(dev), cache()
    torch.cuda.set_sync_debug_mode("error")  # a blocking copy raises
    try:
        outs = calls(c, rows)
        assert c.attend([], rows[2][:0]).shape == (0, H, D)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    compare(outs, rows)


def test_calls_return_while_the_stream_is_busy(dev):
    """All calls are enqueued behind work that is still running, and see their own
    numbers when they run, not those of later calls."""
    rows = inputs(dev)
    compare(calls(cache(), rows), rows)  # memory is there before the clock runs
    c = cache()
    torch.cuda.synchronize()
    torch.cuda._sleep(100_000_000)       # some tens of milliseconds or more
    done = torch.cuda.Event()
    done.record()
    outs = calls(c, rows)
    assert not done.query(), "a call waited for the stream"
    compare(outs, rows)


def test_calls_cannot_be_captured(dev):
    """They hold the host's numbers of one step; refused before anything has changed."""
    rows, c = inputs(dev), cache()
    a = c.add()
    c.append([a], [3], rows[0][:3], rows[1][:3])
    want = c.attend([a], rows[2][:1])
    free = c.free_pages
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = rows[2] + 0
        with pytest.raises(RuntimeError, match="captured"):
            c.append([a], [9], rows[0][:9], rows[1][:9])
        with pytest.raises(RuntimeError, match="captured"):
            c.attend([a], rows[2][:1])
    graph.replay()
    assert torch.equal(held, rows[2])
    assert (c.length(a), c.free_pages) == (3, free)
    assert torch.equal(c.attend([a], rows[2][:1]), want)


def test_on_another_stream(dev):
    rows = inputs(dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = calls(cache(), rows)
    torch.cuda.current_stream().wait_stream(side)
    compare(outs, rows)

"""Rotation, 4-bit caches and their attention as they are used together: a prompt
trained on and served, sessions behind a cached history, captured and on other
streams, through the cache object."""

import numpy as np
import pytest
import torch

from attention_helpers import attention, check
from mx_fbgemm.sequence_attention import PagedSequenceCache, rotary_table
from rows_helpers import angles, attention4, make, rotate, rows4, values4

pytestmark = pytest.mark.gpu

OPS = torch.ops.mx_fbgemm
H, Hkv, D = 4, 2, 64


def cache(bits, dtype=torch.bfloat16, rotary=True, interleaved=False, **kw):
    args = dict(pages=64, page_size=16, heads=Hkv, head_dim=D, max_sequences=4, max_length=200)
    return PagedSequenceCache(**{**args, **kw}, dtype=dtype, bits=bits, interleaved=interleaved,
                              rotary=rotary_table(200, D) if rotary else None)


def turned(x, first, interleaved=False):
    """One list's rows [n, h, D], the first at position `first`, turned in fp32."""
    return rotate(x, [0, x.shape[0]], angles(200, D), [first], interleaved)


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_prompts_then_single_events(dev, bits, interleaved, dtype):
    """Prompts, then single events: each output is attention over all of the
    sequence's rows so far, as the cache holds them."""
    dt = getattr(torch, dtype)
    c = cache(bits, dt, interleaved=interleaved)
    names = [c.add() for _ in range(3)]
    counts = [37, 1, 120]
    rows = {s: [torch.zeros((0, Hkv, D))] * 2 for s in names}

    def append(who, n, seed):
        q, k, v = (make((sum(n), h, D), dtype, seed + i) for i, h in enumerate((H, Hkv, Hkv)))
        at, want = 0, []
        for s, m in zip(who, n):
            first = rows[s][0].shape[0]
            want.append(turned(q[at:at + m], first, interleaved))
            kr = turned(k[at:at + m], first, interleaved)
            rows[s] = [torch.cat([rows[s][0], kr]), torch.cat([rows[s][1], v[at:at + m].float()])]
            at += m
        out = c.append(who, n, k.to(dev), v.to(dev), q.to(dev))
        assert torch.equal(out.cpu(), torch.cat(want).to(dt))
        return out

    append(names, counts, 1)
    for step in range(3):
        who = [names[2], names[0], names[1]] if step else names
        q = append(who, [1] * 3, 10 + step)
        got = c.attend(who, q).double().cpu().numpy()
        qn = q.double().cpu().numpy()
        if bits == 4:
            want, tol = attention4(qn, [rows4(rows[s][0]) for s in who], [rows4(rows[s][1]) for s in who], D ** -0.5, dtype)
        else:
            parts = [attention(qn[i:i + 1], rows[s][0].to(dt).double().numpy(), rows[s][1].to(dt).double().numpy(), [0, 1],
                               [0, rows[s][0].shape[0]], False, D ** -0.5, dtype) for i, s in enumerate(who)]
            want, tol = np.concatenate([p.out for p in parts]), np.concatenate([p.out_tol for p in parts])
        check(got, want, tol, f"step {step}")


@pytest.mark.parametrize("bits", [4, 16])
def test_a_session_behind_its_history(dev, bits):
    """Several new events: what gather gives goes into jagged_attention with the
    new events' queries, and agrees with the float64 definition on those rows."""
    c = cache(bits)
    names = [c.add(), c.add()]
    hist, new = [50, 3], [7, 1]
    for n, seed in ((hist, 1), (new, 5)):
        q, k, v = (make((sum(n), h, D), "bfloat16", seed + i) for i, h in enumerate((H, Hkv, Hkv)))
        q = c.append(names, n, k.to(dev), v.to(dev), q.to(dev))
    k, v, offsets = c.gather(names)
    assert offsets.tolist() == [0, 57, 61] and k.shape == (61, Hkv, D) and k.dtype == torch.bfloat16
    qo = torch.tensor([0, 7, 8], device=dev, dtype=torch.int32)
    out = OPS.jagged_attention(q, k, v, qo, offsets)
    want = attention(q.double().cpu().numpy(), k.double().cpu().numpy(), v.double().cpu().numpy(), [0, 7, 8], [0, 57, 61],
                     True, D ** -0.5, "bfloat16")
    check(out.double().cpu().numpy(), want.out, want.out_tol, "out")
    # A sequence that has left leaves the others' rows where they are.
    before = c.gather([names[1]])[0].clone()
    c.remove(names[0])
    assert torch.equal(c.gather([names[1]])[0], before)
    assert c.gather([])[0].shape == (0, Hkv, D)


def test_training_and_serving_agree(dev):
    """The last event of every list: jagged_rotary and jagged_attention over whole
    lists, against the same rows served from a 16-bit rotating cache.  Both round
    rotated rows to bf16 alike, so they attend over the same bits; each is within
    its own bound of the definition."""
    lengths = [40, 1, 90]
    off = np.concatenate([[0], np.cumsum(lengths)])
    q, k, v = (make((off[-1], h, D), "bfloat16", i).to(dev) for i, h in enumerate((H, Hkv, Hkv)))
    o, table = torch.from_numpy(off).to(dev), rotary_table(200, D)
    qk = OPS.jagged_rotary(torch.cat([q, k], 1), o, table)
    whole = OPS.jagged_attention(qk[:, :H], qk[:, H:], v, o)
    c = cache(16)
    names = [c.add() for _ in lengths]
    qs = c.append(names, lengths, k, v, q)
    assert torch.equal(qs, qk[:, :H])
    got = c.attend(names, qs[off[1:] - 1])
    r = attention(qk[:, :H].double().cpu().numpy(), qk[:, H:].double().cpu().numpy(), v.double().cpu().numpy(), off, off,
                  True, D ** -0.5, "bfloat16")
    check(whole.double().cpu().numpy(), r.out, r.out_tol, "whole")
    check(got.double().cpu().numpy(), r.out[off[1:] - 1], r.out_tol[off[1:] - 1], "served")


def test_gradients_through_rotation_and_attention(dev):
    """The whole path's gradients against plain fp32 autograd: values of order 1, a
    few bf16 roundings (2^-8) one after another."""
    off = torch.tensor([0, 9, 9, 30], device=dev)
    q, k, v, g = (make((30, h, D), "bfloat16", i).to(dev) for i, h in enumerate((H, Hkv, Hkv, H)))
    table = rotary_table(64, D)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    out = OPS.jagged_attention(OPS.jagged_rotary(leaves[0], off, table), OPS.jagged_rotary(leaves[1], off, table), leaves[2], off)
    grads = torch.autograd.grad(out, leaves, g)
    plain = [x.double().cpu().requires_grad_() for x in (q, k, v)]
    outs = []
    t = angles(64, D).double()
    for a, b in ((0, 9), (9, 30)):
        n = b - a
        qr, kr = (torch.cat([x[a:b, :, :32] * t[:n, None, :, 0] - x[a:b, :, 32:] * t[:n, None, :, 1],
                             x[a:b, :, 32:] * t[:n, None, :, 0] + x[a:b, :, :32] * t[:n, None, :, 1]], -1) for x in plain[:2])
        for h in range(H):
            s = qr[:, h] @ kr[:, h // 2].T / 8
            s = s.masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), float("-inf"))
            outs.append((a, h, torch.softmax(s, -1) @ plain[2][a:b, h // 2]))
    want = torch.stack([torch.cat([o for a, hh, o in outs if hh == h]) for h in range(H)], 1)
    wants = torch.autograd.grad(want, plain, g.double().cpu())
    for got, ref in zip((out.detach(), *grads), (want.detach(), *wants)):
        torch.testing.assert_close(got.double().cpu(), ref, rtol=3e-2, atol=6e-2)


@pytest.mark.parametrize("bits", [4, 16])
def test_a_serving_step_in_a_graph(dev, bits):
    """Append (rotating), attention and gather captured once; replays with other
    numbers on the device, between them eager work, each checked against eager."""
    page, B, width = 16, 5, 8
    shape = (B * width, page, Hkv, D // 2 + 4 if bits == 4 else D)
    kc, vc = (torch.zeros(shape, dtype=torch.uint8 if bits == 4 else torch.bfloat16, device=dev) for _ in range(2))
    table = torch.arange(B * width, dtype=torch.int32, device=dev).view(B, width)
    t = rotary_table(200, D)
    off, starts = torch.arange(B + 1, device=dev), torch.zeros(B, dtype=torch.int64, device=dev)
    lengths, all_off = torch.ones(B, dtype=torch.int64, device=dev), torch.arange(B + 1, device=dev)
    q, k, v = (torch.zeros((B, h, D), dtype=torch.bfloat16, device=dev) for h in (H, Hkv, Hkv))

    def step():
        qr = OPS.paged_cache_append_rotary(q, k, v, off, starts, t, kc, vc, table)
        return (qr, OPS.paged_cache_attention(qr, kc, vc, table, lengths),
                *OPS.paged_cache_gather(kc, vc, table, all_off, 200, torch.bfloat16))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(6):
        for x, h in ((q, H), (k, Hkv), (v, Hkv)):
            x.copy_(make((B, h, D), "bfloat16", 10 * i + h))
        starts.fill_(i * 7), lengths.fill_(i * 7 + 1), all_off.copy_(torch.arange(B + 1) * (i * 7 + 1))
        kc0, vc0 = kc.clone(), vc.clone()
        graph.replay()
        got = [x.clone() for x in outs]
        kc1, vc1 = kc.clone(), vc.clone()
        kc.copy_(kc0), vc.copy_(vc0)
        torch.cuda.synchronize()
        want = step()
        assert torch.equal(kc, kc1) and torch.equal(vc, vc1)
        for a, b in zip(got, want):
            assert torch.equal(a, b), i


def test_two_streams_at_once(dev):
    """Two caches on two streams, with workspaces of their own (long sequences in shares)."""
    args = []
    for seed in (1, 2):
        rows = rows4(make((200, 16, 1, D), torch.float32, seed)).to(dev)
        table = torch.randperm(200, generator=torch.Generator().manual_seed(seed)).int().view(2, 100).to(dev)
        args.append((make((2, 8, D), "float16", seed).to(dev), rows, rows, table, torch.tensor([1600, 1234], device=dev)))
    want = [OPS.paged_cache_attention(*a) for a in args]
    streams = [torch.cuda.Stream() for _ in args]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, a in zip(streams, args):
            with torch.cuda.stream(s):
                got.append(OPS.paged_cache_attention(*a))
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_four_bits_against_sixteen(dev):
    """The same events in both caches: what differs is the rounding of the rows, half
    a step (a thirtieth of a row's range) at most, and scale's and bias's in fp16."""
    c4, c16 = cache(4), cache(16)
    k, v, q = (make((100, h, D), "bfloat16", i).to(dev) for i, h in enumerate((Hkv, Hkv, H)))
    for c in (c4, c16):
        c.append([c.add()], [100], k, v, q)
    for a, b in zip(c4.gather([0])[:2], c16.gather([0])[:2]):
        a, b = a.float(), b.float()
        span = b.amax(-1, keepdim=True) - b.amin(-1, keepdim=True)
        largest = b.abs().amax(-1, keepdim=True)
        # 16-bit rows, and 4-bit ones read back, are rounded to bf16 (2^-8) too.
        assert ((a - b).abs() <= span * (1 / 30 + 2 * 2 ** -8) + largest * (16 * 2.0 ** -11 + 2 * 2.0 ** -8)).all()


def test_no_call_synchronizes(dev):
    c = cache(4)
    a = c.add()
    k, q = make((30, Hkv, D), "bfloat16", 1).to(dev), make((30, H, D), "bfloat16", 2).to(dev)
    c.append([a], [30], k, k, q)
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        q = c.append([a], [30], k, k, q)
        c.attend([a], q[:1])
        c.gather([a])
    finally:
        torch.cuda.set_sync_debug_mode("default")
    with pytest.raises(RuntimeError, match="captured"):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.gather([a])


def test_append_without_queries_or_rotation(dev):
    c = cache(4, rotary=False)
    a = c.add()
    k, q = make((5, Hkv, D), "bfloat16", 1).to(dev), make((5, H, D), "bfloat16", 2).to(dev)
    assert c.append([a], [5], k, k) is None
    assert c.append([a], [5], k, k, q) is q
    got = c.gather([a])[0].cpu()
    want = torch.from_numpy(values4(rows4(k.cpu()))).float().bfloat16()
    assert torch.equal(got, torch.cat([want, want]))
    c = cache(16)
    assert c.append([c.add()], [5], k, k) is None

"""Performance cases of positions, and of a key-value cache held in 4 bits.

A sequence model that knows its events' positions rotates queries and keys by
them, in training and, on the way into the cache, in serving; a cache of four
bits a value holds almost four times the events.  The cases:

* ``rotate``: rotation of packed queries and keys, with its gradient;
* ``append``: a batch's new events into a 16-bit paged cache, rotated on the way;
* ``chunk``: new events into a paged cache (4 or 16 bits), rotated on the way,
  and every list's keys and values out of it again, packed: what attention over
  a cached history and several new events takes;
* ``step``: attention of one new event per user over a 4-bit cache.

A row of a 4-bit cache is the head's codes, two to a byte (the even element in
the low half), then scale and bias in fp16: value = scale * code + bias.

``run`` computes each in its plain form (elementary torch operations, in 32
bits) or, where ``own`` is set, by this package's operators.
"""

from __future__ import annotations

import math
import random
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}
INDEX = {"int32": torch.int32, "int64": torch.int64}


def listed() -> list[dict]:
    return [
        # A training step on a small local batch of sessions.
        dict(name="rotate_small", kind="rotate", B=8, L=64, extra=0, lengths="uniform", H=4, Hkv=4,
             D=64, R=64, interleaved=False, dtype="float16", index="int64", fused=False),
        # A training batch of user histories, long-tailed; queries and keys lie
        # in one projection's output.
        dict(name="rotate_batch", kind="rotate", B=256, L=512, extra=0, lengths="log", H=8, Hkv=8,
             D=96, R=96, interleaved=True, dtype="bfloat16", index="int32", fused=True),
        # Training on long histories; half of each head carries positions.
        dict(name="rotate_long", kind="rotate", B=4, L=4096, extra=0, lengths="fixed", H=16, Hkv=4,
             D=128, R=64, interleaved=False, dtype="bfloat16", index="int64", fused=True),
        # One new event per user into the cache.
        dict(name="append_step", kind="append", bits=16, B=64, L=1, extra=4096, lengths="fixed",
             page=16, H=32, Hkv=8, D=128, R=128, interleaved=False, dtype="bfloat16", index="int32"),
        # Whole histories into the cache, in the pass that rotates them.
        dict(name="append_prompt", kind="append", bits=16, B=32, L=2000, extra=0, lengths="uniform",
             page=64, H=16, Hkv=8, D=128, R=128, interleaved=False, dtype="bfloat16", index="int64"),
        # One new event per user behind short sessions, in 4 bits.
        dict(name="chunk_small", kind="chunk", bits=4, B=64, L=1, extra=40, lengths="fixed", page=16,
             H=8, Hkv=8, D=64, R=64, interleaved=False, dtype="float16", index="int32"),
        # A session's new events behind a cached history.
        dict(name="chunk_history", kind="chunk", bits=4, B=16, L=250, extra=2000, lengths="uniform",
             page=16, H=8, Hkv=8, D=128, R=128, interleaved=True, dtype="bfloat16", index="int64"),
        # The same from a 16-bit cache.
        dict(name="chunk_history16", kind="chunk", bits=16, B=16, L=250, extra=2000,
             lengths="uniform", page=16, H=8, Hkv=8, D=128, R=128, interleaved=False,
             dtype="float16", index="int32"),
        # One user's next event: a single short list.
        dict(name="step_small", kind="step", bits=4, B=1, L=777, lengths="fixed", page=16, H=8, Hkv=8,
             D=64, dtype="bfloat16", index="int32"),
        # The next event of a batch of users whose histories differ widely.
        dict(name="step_batch", kind="step", bits=4, B=64, L=4096, lengths="uniform", page=16, H=32,
             Hkv=8, D=128, dtype="bfloat16", index="int32"),
        # A large serving batch over long caches: memory bound throughout.
        dict(name="step_large", kind="step", bits=4, B=256, L=8192, lengths="fixed", page=64, H=16,
             Hkv=4, D=128, dtype="float16", index="int64"),
    ]


#: Bounds of the drawn cases, at most the largest listed ones: elements of
#: queries and keys (rotate), of all three appended tensors, of keys read back,
#: of a cache.
MOST = {"rotate": 4 * 4096 * 20 * 128, "append": 32 * 1000 * 32 * 128,
        "chunk": 16 * 1125 * 8 * 128, "step": 256 * 8192 * 4 * 128}


def _log(rng: random.Random, lo: float, hi: float) -> int:
    return max(1, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi)))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["rotate", "rotate", "append", "chunk", "chunk", "step", "step", "step"])
    D = rng.choice([32, 40, 64, 64, 80, 96, 128, 128])
    Hkv = rng.choice([1, 2, 4, 8])
    H = Hkv * rng.choice([g for g in (1, 2, 4, 8) if Hkv * g <= 32])
    c = dict(kind=kind, lengths=rng.choice(["fixed", "uniform", "log"]), H=H, Hkv=Hkv, D=D,
             dtype=rng.choice(list(DTYPES)), index=rng.choice(list(INDEX)))
    if kind != "rotate":
        c.update(page=rng.choice([8, 16, 32, 64, 128]))
    if kind == "step":
        L = _log(rng, 2, 131072)
        return dict(c, bits=4, L=L, B=_log(rng, 1, min(256, MOST[kind] / (L * Hkv * D))))
    c.update(R=rng.choice([D, D, D, D // 16 * 8]), interleaved=rng.random() < 0.5)
    if kind == "rotate":
        L = _log(rng, 2, 4096)
        return dict(c, L=L, extra=rng.choice([0, 0, _log(rng, 1, 4096)]), fused=rng.random() < 0.5,
                    B=_log(rng, 1, min(256, MOST[kind] / ((H + Hkv) * L * D))))
    L, extra = rng.choice([1, _log(rng, 1, 2000)]), rng.choice([0, _log(rng, 1, 4096)])
    if kind == "append":
        return dict(c, bits=16, L=L, extra=extra,
                    B=_log(rng, 1, min(512, MOST[kind] / (L * (H + 2 * Hkv) * D),
                                       MOST[kind] / ((L + extra) * Hkv * D))))
    return dict(c, bits=rng.choice([4, 4, 16]), L=min(L, 500), extra=extra,
                B=_log(rng, 1, min(512, MOST[kind] / ((min(L, 500) + extra) * Hkv * D))))


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _lengths(case: dict) -> np.ndarray:
    """The lists' (new) lengths: the quantiles of their distribution (the seed
    only orders them, so that a case's work is one number).  Of ten or more
    lists that are not all alike, the shortest tenth is empty."""
    B, L = case["B"], case["L"]
    u = (np.arange(B) + 0.5) / B
    if case["lengths"] == "fixed":
        return np.full(B, L, np.int64)
    n = np.ceil(u * L) if case["lengths"] == "uniform" else np.round(np.exp(u * math.log(L)))
    n = np.clip(n, 1, L).astype(np.int64)
    n[-1] = L
    if B >= 10 and case["kind"] != "step":
        n[: B // 10] = 0
    return n


def _before(case: dict, n: np.ndarray) -> np.ndarray:
    """Events of each list before its first new one."""
    e = case.get("extra", 0)
    return (np.arange(n.size) * 7919 % (e + 1) if e else np.zeros(n.size, np.int64)).astype(np.int64)


def _offsets(n: np.ndarray, index: str) -> torch.Tensor:
    o = np.zeros(n.size + 1, np.int64)
    np.cumsum(n, out=o[1:])
    return torch.from_numpy(o).to(DEV).to(INDEX[index])


def _randn(shape, dtype, gen):
    return torch.randn(shape, dtype=torch.float32, device=DEV, generator=gen).to(dtype)


def _angles(positions: int, R: int) -> torch.Tensor:
    """[positions, R / 2] angles in 64 bits: position * 10000 ** (-2 i / R)."""
    i = torch.arange(R // 2, dtype=torch.float64, device=DEV)
    return torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * 10000.0 ** (-2 * i / R)


def _rows4(values: torch.Tensor) -> torch.Tensor:
    """[..., D] fp32 values as rows of a 4-bit cache, [..., D / 2 + 4] bytes."""
    low, high = values.amin(-1, keepdim=True), values.amax(-1, keepdim=True)
    bias = low.half()
    spread = high - bias.float()
    scale = torch.where(spread == 0, torch.ones_like(spread), spread / 15.0).half()
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    codes = ((values - bias.float()) * (1.0 / scale.float())).round().clamp(0, 15).to(torch.uint8)
    tail = torch.cat([scale, bias], -1).contiguous().view(torch.uint8)
    return torch.cat([codes[..., 0::2] | (codes[..., 1::2] << 4), tail], -1)


def _cache(case: dict, pages: int, gen) -> torch.Tensor:
    """A cache in use: [pages, page, Hkv, D], or rows of 4 bits, whose pages
    hold each head's rows together."""
    dt, page, Hkv, D = DTYPES[case["dtype"]], case["page"], case["Hkv"], case["D"]
    if case["bits"] == 16:
        return torch.empty((pages, page, Hkv, D), dtype=dt, device=DEV).normal_(generator=gen)
    rows = torch.empty((pages, Hkv, page, D // 2 + 4), dtype=torch.uint8, device=DEV)
    some = max(1, (1 << 26) // (page * Hkv * D))
    for p in range(0, pages, some):
        part = rows[p: p + some]
        part.copy_(_rows4(torch.randn((*part.shape[:3], D), device=DEV, generator=gen)))
    return rows.transpose(1, 2)


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rng = np.random.default_rng(seed)
    n, dt = _lengths(case), DTYPES[case["dtype"]]
    order = rng.permutation(n.size)
    H, Hkv, D = case["H"], case["Hkv"], case["D"]
    before = _before(case, n)[order]
    n = n[order]
    total = n + before
    N = int(n.sum())
    s = dict(case=case)
    if case["kind"] != "step":
        angles = _angles(int(total.max()) + 1, case["R"])
        s["rotary"] = torch.stack([angles.cos(), angles.sin()], -1).float()
        s["offsets"] = _offsets(n, case["index"])
        s["starts"] = torch.from_numpy(before).to(DEV).to(INDEX[case["index"]])
    if case["kind"] == "rotate":
        x = _randn((N, H + (2 if case["fused"] else 1) * Hkv, D), dt, gen)
        s["x"] = x[:, :H + Hkv].detach().requires_grad_()
        s["grad"] = _randn((N, H + Hkv, D), dt, gen)
        return s
    page = case["page"]
    pages = -(-total // page)
    width = max(1, int(pages.max()))
    # Pages come from a pool in no order; what a list does not use is -1.
    pool = rng.permutation(int(pages.sum()) + 8).astype(np.int32)
    table = np.full((n.size, width), -1, np.int32)
    table[np.arange(width)[None, :] < pages[:, None]] = pool[: int(pages.sum())]
    s.update(table=torch.from_numpy(table).to(DEV), k_cache=_cache(case, pool.size, gen),
             v_cache=_cache(case, pool.size, gen))
    if case["kind"] == "step":
        s.update(q=_randn((n.size, H, D), dt, gen), scale=1.0 / math.sqrt(D),
                 lengths=torch.from_numpy(total).to(DEV).to(INDEX[case["index"]]))
        return s
    x = _randn((N, H + 2 * Hkv, D), dt, gen)
    s.update(q=x[:, :H], k=x[:, H:H + Hkv], v=x[:, H + Hkv:])
    if case["kind"] == "chunk":
        s.update(total=int(total.sum()), all_offsets=_offsets(total, case["index"]))
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

_loaded = None


def _ops():
    global _loaded
    if _loaded is None:
        sys.path.insert(0, "torchlib-xpu_amd")
        import mx_fbgemm  # noqa: F401  (registers torch.ops.mx_fbgemm.*)

        _loaded = torch.ops.mx_fbgemm
    return _loaded


def run(s: dict):
    return {"rotate": _rotate, "append": _append, "chunk": _chunk, "step": _step}[s["case"]["kind"]](s)


def _list_of_row(offsets, N):
    """The list that holds each of N rows."""
    return torch.searchsorted(offsets, torch.arange(N, device=DEV, dtype=offsets.dtype), right=True) - 1


def _positions(s, N):
    """Each row's list, and its position."""
    o = s["offsets"].long()
    b = _list_of_row(o, N)
    return b, s["starts"].long()[b] + torch.arange(N, device=DEV) - o[b]


def _rotated(x, at, rotary, interleaved, sign=1.0):
    """x [N, H, D] in 32 bits, its first columns rotated by the angles of positions `at`."""
    R = 2 * rotary.size(1)
    c, t = rotary[at][:, None, :, 0], rotary[at][:, None, :, 1] * sign
    x = x.float()
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    u, w = a * c - b * t, b * c + a * t
    both = torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1)
    return torch.cat([both, x[..., R:]], -1)


def _rotate(s):
    c, x = s["case"], s["x"]
    if own:
        y = _ops().jagged_rotary(x, s["offsets"], s["rotary"], s["starts"], c["interleaved"])
        return (y.detach(), *torch.autograd.grad(y, (x,), s["grad"]))
    with torch.no_grad():
        _, at = _positions(s, x.size(0))
        return (_rotated(x, at, s["rotary"], c["interleaved"]).to(x.dtype),
                _rotated(s["grad"], at, s["rotary"], c["interleaved"], -1.0).to(x.dtype))


def _append(s):
    c, kc, vc = s["case"], s["k_cache"], s["v_cache"]
    if own:
        q = _ops().paged_cache_append_rotary(s["q"], s["k"], s["v"], s["offsets"], s["starts"],
                                             s["rotary"], kc, vc, s["table"], c["interleaved"])
        return q, kc, vc
    page = c["page"]
    b, at = _positions(s, s["k"].size(0))
    pages = s["table"].long()[b, at // page]
    k, v = _rotated(s["k"], at, s["rotary"], c["interleaved"]), s["v"]
    kc[pages, at % page] = _rows4(k) if c["bits"] == 4 else k.to(kc.dtype)
    vc[pages, at % page] = _rows4(v.float()) if c["bits"] == 4 else v
    return _rotated(s["q"], at, s["rotary"], c["interleaved"]).to(s["q"].dtype), kc, vc


def _values4(rows):
    """The fp32 values of rows of a 4-bit cache."""
    codes = rows[..., :-4]
    tail = rows[..., -4:].contiguous().view(torch.float16).float()
    x = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    return x * tail[..., :1] + tail[..., 1:]


def _chunk(s):
    c = s["case"]
    q, kc, vc = _append(s)
    dt, page = s["k"].dtype, c["page"]
    if own:
        return (q, *_ops().paged_cache_gather(kc, vc, s["table"], s["all_offsets"], s["total"], dt))
    o = s["all_offsets"].long()
    b = _list_of_row(o, s["total"])
    at = torch.arange(s["total"], device=DEV) - o[b]
    pages = s["table"].long()[b, at // page]
    k, v = kc[pages, at % page], vc[pages, at % page]
    return (q, _values4(k).to(dt), _values4(v).to(dt)) if c["bits"] == 4 else (q, k, v)


def _step(s):
    c = s["case"]
    if own:
        return _ops().paged_cache_attention(s["q"], s["k_cache"], s["v_cache"], s["table"],
                                            s["lengths"], s["scale"])
    B, H, Hkv, D = c["B"], c["H"], c["Hkv"], c["D"]
    pages = s["table"].long().clamp(min=0)
    k = _values4(s["k_cache"][pages]).view(B, -1, Hkv, D).permute(0, 2, 3, 1)
    q = s["q"].float().view(B, Hkv, H // Hkv, D)
    p = torch.matmul(q, k).mul_(s["scale"])
    del k
    see = torch.arange(p.size(3), device=DEV)[None, :] < s["lengths"][:, None]
    p.masked_fill_(~see[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    v = _values4(s["v_cache"][pages]).view(B, -1, Hkv, D).permute(0, 2, 1, 3)
    o = torch.matmul(p, v).div_(torch.where(total == 0, 1.0, total))
    return o.view(B, H, D).to(s["q"].dtype)


# ---------------------------------------------------------------------------
# Work and the definition in 64 bits
# ---------------------------------------------------------------------------

def work(case: dict) -> dict:
    n = _lengths(case)
    before = _before(case, n)
    N, all_, H, Hkv, D = int(n.sum()), int((n + before).sum()), case["H"], case["Hkv"], case["D"]
    row = D // 2 + 4 if case.get("bits") == 4 else 2 * D  # bytes in a cache
    if case["kind"] == "step":
        return {"bytes": 2 * all_ * Hkv * row + 2 * n.size * H * D * 2, "flops": 4 * D * H * all_}
    angles = 4 * case["R"] * int((n + before).max())
    turned = 3 * case["R"] * N * (H + Hkv)
    if case["kind"] == "rotate":
        return {"bytes": 4 * 2 * D * N * (H + Hkv) + angles, "flops": 2 * turned}
    new = 2 * D * N * (2 * H + 2 * Hkv) + 2 * N * Hkv * row + angles
    if case["kind"] == "append":
        return {"bytes": new, "flops": turned}
    return {"bytes": new + 2 * all_ * Hkv * (row + 2 * D), "flops": turned}


def _numbers(row: np.ndarray) -> np.ndarray:
    """What 4-bit rows ([..., D / 2 + 4] bytes) stand for, in 64 bits."""
    out = np.empty((*row.shape[:-1], 2 * (row.shape[-1] - 4)))
    ends = np.ascontiguousarray(row[..., -4:]).view(np.float16).astype(np.float64)
    out[..., 0::2], out[..., 1::2] = row[..., :-4] % 16, row[..., :-4] // 16
    return out * ends[..., 0, None] + ends[..., 1, None]


def _through4(x: np.ndarray) -> np.ndarray:
    """Values x [..., D] as a 4-bit row gives them back, in 64 bits."""
    bias = x.min(-1, keepdims=True).astype(np.float16).astype(np.float64)
    step = ((x.max(-1, keepdims=True) - bias) / 15).astype(np.float16).astype(np.float64)
    step[step == 0] = 1.0
    return np.clip(np.rint((x - bias) / step), 0, 15) * step + bias


def _turn(x: np.ndarray, first: int, case: dict, sign: float = 1.0) -> np.ndarray:
    """x [n, H, D] of one list, its first row at position `first`, as complex numbers."""
    R = case["R"]
    w = 10000.0 ** (-2 * np.arange(R // 2) / R)
    z = np.exp(1j * sign * (first + np.arange(x.shape[0]))[:, None] * w)[:, None]
    y = x.copy()
    if case["interleaved"]:
        z = z * (x[..., 0:R:2] + 1j * x[..., 1:R:2])
        y[..., 0:R:2], y[..., 1:R:2] = z.real, z.imag
    else:
        z = z * (x[..., :R // 2] + 1j * x[..., R // 2:R])
        y[..., :R // 2], y[..., R // 2:R] = z.real, z.imag
    return y


def exact(case: dict, seed: int):
    """The same outputs list by list in 64 bits."""
    s = prepare(case, seed)
    kind, page = case["kind"], case.get("page", 1)

    def array(x):
        return x.detach().to(torch.float64).cpu().numpy()

    if kind == "step":
        B, H, Hkv, D = case["B"], case["H"], case["Hkv"], case["D"]
        out = torch.zeros((B, H, D), dtype=torch.float64, device=DEV)
        G = H // Hkv
        for b, n in enumerate(s["lengths"].tolist()):
            pages = s["table"][b, : -(-n // page)].long()
            for h in range(Hkv):
                kv = []
                for cache in (s["k_cache"], s["v_cache"]):
                    r = cache[pages, :, h].reshape(-1, D // 2 + 4)[:n]
                    ends = r[:, -4:].contiguous().view(torch.float16).double()
                    x = torch.empty((n, D), dtype=torch.float64, device=DEV)
                    x[:, 0::2], x[:, 1::2] = (r[:, :-4] & 15).double(), (r[:, :-4] >> 4).double()
                    kv.append(x * ends[:, :1] + ends[:, 1:])
                w = torch.softmax(s["q"][b, h * G:(h + 1) * G].double() @ kv[0].T * s["scale"], dim=-1)
                out[b, h * G:(h + 1) * G] = w @ kv[1]
        return out
    o, starts = s["offsets"].tolist(), s["starts"].tolist()
    lists = [(slice(o[b], o[b + 1]), starts[b]) for b in range(case["B"])]
    if kind == "rotate":
        x, g = array(s["x"]), array(s["grad"])
        y, d = np.empty_like(x), np.empty_like(g)
        for rows, first in lists:
            y[rows], d[rows] = _turn(x[rows], first, case), _turn(g[rows], first, case, -1.0)
        return torch.from_numpy(y), torch.from_numpy(d)
    q, k, v = (array(s[name]) for name in ("q", "k", "v"))
    for rows, first in lists:
        q[rows], k[rows] = _turn(q[rows], first, case), _turn(k[rows], first, case)
    table = s["table"].cpu().numpy()
    if kind == "append":
        kc, vc = array(s["k_cache"]), array(s["v_cache"])
        for b, (rows, first) in enumerate(lists):
            t = first + np.arange(rows.stop - rows.start)
            kc[table[b, t // page], t % page] = k[rows]
            vc[table[b, t // page], t % page] = v[rows]
        return torch.from_numpy(q), torch.from_numpy(kc), torch.from_numpy(vc)
    four = case["bits"] == 4
    if four:
        kc, vc = s["k_cache"].cpu().numpy(), s["v_cache"].cpu().numpy()
    else:
        kc, vc = array(s["k_cache"]), array(s["v_cache"])
    got = [[], []]
    for b, (rows, first) in enumerate(lists):
        t = np.arange(first)
        for cache, new, to in ((kc, k, got[0]), (vc, v, got[1])):
            old = cache[table[b, t // page], t % page]
            to += [_numbers(old), _through4(new[rows])] if four else [old, new[rows]]
    return tuple(torch.from_numpy(x) for x in (q, np.concatenate(got[0]), np.concatenate(got[1])))

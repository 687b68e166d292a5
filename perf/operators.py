"""Performance cases of attention over jagged sequences and its paged cache.

The sequence lookups of this package give one row per event together with the
batch's offsets.  These cases are what a model does with such rows next:

* ``prompt``: attention over packed sequences (every user's history in one
  tensor, cut by offsets), causal, with grouped key-value heads;
* ``train``: the same with its gradients;
* ``append``: writing the keys and values of new events into a paged cache;
* ``step``: attention of one new event per user over that cache.

``run`` computes each in its plain form (elementary torch operations on padded
tensors, in 32 bits) or, where ``own`` is set, by this package's operators.
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
        # One small request batch: a handful of short histories, where the
        # call's latency is all there is.
        dict(name="prompt_small", kind="prompt", B=4, L=40, extra=0, lengths="uniform", causal=True,
             H=4, Hkv=4, D=32, dtype="bfloat16", index="int64", fused=False),
        # The histories of an ordinary scoring batch, ragged, some empty.
        dict(name="prompt_batch", kind="prompt", B=64, L=1000, extra=0, lengths="uniform",
             causal=True, H=8, Hkv=2, D=64, dtype="float16", index="int64", fused=True),
        # Life-long histories: few lists, thousands of events each.
        dict(name="prompt_long", kind="prompt", B=2, L=8192, extra=0, lengths="fixed", causal=True,
             H=16, Hkv=4, D=128, dtype="bfloat16", index="int64", fused=True),
        # A session's new events attending to the session and the history
        # before it: more keys than queries.
        dict(name="prompt_history", kind="prompt", B=16, L=250, extra=2000, lengths="uniform",
             causal=True, H=8, Hkv=8, D=128, dtype="bfloat16", index="int32", fused=False),
        # A training step's attention on a small local batch.
        dict(name="train_small", kind="train", B=8, L=64, extra=0, lengths="uniform", causal=True,
             H=4, Hkv=4, D=64, dtype="float16", index="int64", fused=False),
        # A training batch of user histories, long-tailed, head width that is
        # no power of two.
        dict(name="train_batch", kind="train", B=256, L=512, extra=0, lengths="log", causal=True,
             H=8, Hkv=8, D=96, dtype="bfloat16", index="int64", fused=True),
        # Training on long histories with shared key-value heads.
        dict(name="train_long", kind="train", B=4, L=4096, extra=0, lengths="fixed", causal=True,
             H=16, Hkv=4, D=128, dtype="bfloat16", index="int64", fused=True),
        # One user's next event: a single short list.
        dict(name="step_small", kind="step", B=1, L=777, lengths="fixed", page=16, H=8, Hkv=8, D=64,
             dtype="bfloat16", index="int32"),
        # The next event of a batch of users whose histories differ widely.
        dict(name="step_batch", kind="step", B=64, L=4096, lengths="uniform", page=16, H=32, Hkv=8,
             D=128, dtype="bfloat16", index="int32"),
        # A large serving batch over long caches: memory bound throughout.
        dict(name="step_large", kind="step", B=256, L=8192, lengths="fixed", page=64, H=16, Hkv=4,
             D=128, dtype="float16", index="int64"),
        # One new event per user into the cache.
        dict(name="append_step", kind="append", B=64, L=1, start=4096, lengths="fixed", page=16,
             Hkv=8, D=128, dtype="bfloat16", index="int32"),
        # Whole histories into the cache, after a prompt.
        dict(name="append_prompt", kind="append", B=32, L=2000, start=0, lengths="uniform", page=64,
             Hkv=8, D=128, dtype="bfloat16", index="int64"),
    ]


#: Bounds of the drawn cases, at most the largest listed ones: scores of a
#: padded batch (prompt; train), elements of a cache (step), rows appended.
MOST = {"prompt": 2 * 16 * 8192 * 8192, "train": 4 * 16 * 4096 * 4096,
        "step": 256 * 8192 * 4 * 128, "append": 32 * 1000 * 8 * 128}


def _log(rng: random.Random, lo: float, hi: float) -> int:
    return max(1, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi)))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["prompt", "prompt", "train", "train", "step", "step", "append"])
    dtype, index = rng.choice(list(DTYPES)), rng.choice(list(INDEX))
    lengths = rng.choice(["fixed", "uniform", "log"])
    D = rng.choice([32, 40, 64, 64, 80, 96, 128, 128])
    Hkv = rng.choice([1, 2, 4, 8])
    if kind in ("prompt", "train"):
        H = Hkv * rng.choice([g for g in (1, 2, 4, 8) if Hkv * g <= 16])
        L = _log(rng, 2, 8192 if kind == "prompt" else 4096)
        extra = rng.choice([0, 0, 0, _log(rng, 1, 4096)])
        B = _log(rng, 1, min(256, MOST[kind] / (H * L * (L + extra)), 262144 / (L + extra)))
        return dict(kind=kind, B=B, L=L, extra=extra, lengths=lengths, causal=rng.random() < 0.8,
                    H=H, Hkv=Hkv, D=D, dtype=dtype, index=index, fused=rng.random() < 0.5)
    page = rng.choice([8, 16, 32, 64, 128])
    if kind == "step":
        L = _log(rng, 2, 131072)
        B = _log(rng, 1, min(256, MOST[kind] / (L * Hkv * D)))
        return dict(kind=kind, B=B, L=L, lengths=lengths, page=page, H=Hkv * rng.choice([1, 2, 4, 8]),
                    Hkv=Hkv, D=D, dtype=dtype, index=index)
    L = rng.choice([1, _log(rng, 1, 4000)])
    B = _log(rng, 1, min(512, MOST[kind] / (L * Hkv * D)))
    return dict(kind=kind, B=B, L=L, start=rng.choice([0, _log(rng, 1, 4096)]), lengths=lengths,
                page=page, Hkv=Hkv, D=D, dtype=dtype, index=index)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _lengths(case: dict) -> np.ndarray:
    """The lists' lengths: the quantiles of their distribution (the seed only
    orders them, so that a case's work is one number).  Of ten or more lists
    that are not all alike, the shortest tenth is empty."""
    B, L = case["B"], case["L"]
    u = (np.arange(B) + 0.5) / B
    if case["lengths"] == "fixed":
        return np.full(B, L, np.int64)
    n = np.ceil(u * L) if case["lengths"] == "uniform" else np.round(np.exp(u * math.log(L)))
    n = np.clip(n, 1, L).astype(np.int64)
    n[-1] = L
    if B >= 10 and case["kind"] in ("prompt", "train"):
        n[: B // 10] = 0
    return n


def _extras(case: dict, n: np.ndarray) -> np.ndarray:
    """Keys before each list's first query."""
    e = case.get("extra", 0)
    return (np.arange(n.size) * 7919 % (e + 1) if e else np.zeros(n.size, np.int64)).astype(np.int64)


def _offsets(n: np.ndarray, index: str) -> torch.Tensor:
    o = np.zeros(n.size + 1, np.int64)
    np.cumsum(n, out=o[1:])
    return torch.from_numpy(o).to(DEV).to(INDEX[index])


def _randn(shape, dtype, gen, scale=1.0):
    return torch.randn(shape, dtype=torch.float32, device=DEV, generator=gen).mul_(scale).to(dtype)


def _rand_cache(shape, dtype, gen):
    x = torch.empty(shape, dtype=dtype, device=DEV)
    return x.normal_(generator=gen)


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rng = np.random.default_rng(seed)
    n = _lengths(case)
    dt = DTYPES[case["dtype"]]
    order = rng.permutation(n.size)
    s = dict(case=case, scale=1.0 / math.sqrt(case["D"]))
    Hkv, D = case["Hkv"], case["D"]
    if case["kind"] in ("prompt", "train"):
        H = case["H"]
        nq, nk = n[order], (n + _extras(case, n))[order]
        Nq, Nk = int(nq.sum()), int(nk.sum())
        if case["fused"] and Nq == Nk:
            # Views of one projection's output.
            x = _randn((Nq, H + 2 * Hkv, D), dt, gen)
            q, k, v = x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
        else:
            q, k, v = (_randn((N, h, D), dt, gen) for N, h in ((Nq, H), (Nk, Hkv), (Nk, Hkv)))
        s.update(q=q, k=k, v=v, q_offsets=_offsets(nq, case["index"]),
                 k_offsets=_offsets(nk, case["index"]), Lq=int(nq.max()), Lk=int(nk.max()))
        if case["kind"] == "train":
            for t in ("q", "k", "v"):
                s[t] = s[t].detach().requires_grad_()
            s["grad"] = _randn((Nq, H, D), dt, gen)
        return s
    page = case["page"]
    n = n[order]
    total = n + case.get("start", 0)
    pages = -(-total // page)
    width = int(pages.max())
    # Pages come from a pool in no order; what a list does not use is -1.
    pool = rng.permutation(int(pages.sum()) + 8).astype(np.int32)
    table = np.full((n.size, width), -1, np.int32)
    table[np.arange(width)[None, :] < pages[:, None]] = pool[: int(pages.sum())]
    s["table"] = torch.from_numpy(table).to(DEV)
    shape = (pool.size, page, Hkv, D)
    if case["kind"] == "step":
        s.update(q=_randn((n.size, case["H"], D), dt, gen), k_cache=_rand_cache(shape, dt, gen),
                 v_cache=_rand_cache(shape, dt, gen),
                 lengths=torch.from_numpy(total).to(DEV).to(INDEX[case["index"]]))
        return s
    N = int(n.sum())
    s.update(k=_randn((N, Hkv, D), dt, gen), v=_randn((N, Hkv, D), dt, gen),
             offsets=_offsets(n, case["index"]),
             starts=torch.from_numpy(total - n).to(DEV).to(INDEX[case["index"]]),
             k_cache=torch.zeros(shape, dtype=dt, device=DEV),
             v_cache=torch.zeros(shape, dtype=dt, device=DEV))
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
    return {"prompt": _prompt, "train": _train, "step": _step, "append": _append}[s["case"]["kind"]](s)


def _list_of_row(offsets, N):
    """The list that holds each of N rows."""
    return (torch.arange(N, device=DEV)[:, None] >= offsets[None, 1:]).sum(1)


def _pad(x, offsets, L):
    """[N, H, D] packed -> [B, H, L, D] in 32 bits, zeros past each list."""
    o = offsets.long()
    at = torch.arange(L, device=DEV)
    inside = at[None, :] < (o[1:] - o[:-1])[:, None]
    rows = (o[:-1, None] + at[None, :]).clamp(max=x.size(0) - 1)
    return torch.where(inside[:, :, None, None], x[rows].float(), 0.0).permute(0, 2, 1, 3)


def _unpad(x, offsets, N, dtype):
    """[B, H, L, D] -> [N, H, D], rounded to `dtype`."""
    o = offsets.long()
    b = _list_of_row(o, N)
    return x[b, :, torch.arange(N, device=DEV) - o[b]].to(dtype)


def _probabilities(s, q, k):
    """Softmax of the visible scores, [B, Hkv, G * Lq, Lk], and q and k padded."""
    c = s["case"]
    B, H, Hkv, D, Lq, Lk = c["B"], c["H"], c["Hkv"], c["D"], s["Lq"], s["Lk"]
    qp = _pad(q, s["q_offsets"], Lq).reshape(B, Hkv, H // Hkv * Lq, D)
    kp = _pad(k, s["k_offsets"], Lk).contiguous()
    p = torch.matmul(qp, kp.transpose(2, 3)).mul_(s["scale"])
    nq, nk = (o[1:] - o[:-1] for o in (s["q_offsets"].long(), s["k_offsets"].long()))
    i, j = torch.arange(Lq, device=DEV)[None, :, None], torch.arange(Lk, device=DEV)[None, None, :]
    see = (i < nq[:, None, None]) & (j < nk[:, None, None])
    if c["causal"]:
        see = see & (j <= i + (nk - nq)[:, None, None])
    p5 = p.view(B, Hkv, H // Hkv, Lq, Lk)
    p5.masked_fill_(~see[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total == 0, 1.0, total))
    return p, qp, kp


def _prompt(s):
    c = s["case"]
    if own:
        return _ops().jagged_attention(s["q"], s["k"], s["v"], s["q_offsets"], s["k_offsets"],
                                       c["causal"], s["scale"])
    p, _, _ = _probabilities(s, s["q"], s["k"])
    o = torch.matmul(p, _pad(s["v"], s["k_offsets"], s["Lk"]).contiguous())
    return _unpad(o.view(c["B"], c["H"], s["Lq"], c["D"]), s["q_offsets"], s["q"].size(0),
                  s["q"].dtype)


def _train(s):
    c = s["case"]
    q, k, v = s["q"], s["k"], s["v"]
    if own:
        out = _ops().jagged_attention(q, k, v, s["q_offsets"], s["k_offsets"], c["causal"],
                                      s["scale"])
        return (out.detach(), *torch.autograd.grad(out, (q, k, v), s["grad"]))
    with torch.no_grad():
        B, H, Hkv, D, Lq, Lk = c["B"], c["H"], c["Hkv"], c["D"], s["Lq"], s["Lk"]
        p, qp, kp = _probabilities(s, q, k)
        vp = _pad(v, s["k_offsets"], Lk).contiguous()
        o = torch.matmul(p, vp)
        do = _pad(s["grad"], s["q_offsets"], Lq).reshape(B, Hkv, H // Hkv * Lq, D)
        dv = torch.matmul(p.transpose(2, 3), do)
        ds = torch.matmul(do, vp.transpose(2, 3))
        ds.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(s["scale"])
        dq = torch.matmul(ds, kp)
        dk = torch.matmul(ds.transpose(2, 3), qp)
        Nq, Nk, dt = q.size(0), k.size(0), q.dtype
        return (_unpad(o.view(B, H, Lq, D), s["q_offsets"], Nq, dt),
                _unpad(dq.view(B, H, Lq, D), s["q_offsets"], Nq, dt),
                _unpad(dk, s["k_offsets"], Nk, dt), _unpad(dv, s["k_offsets"], Nk, dt))


def _step(s):
    c = s["case"]
    if own:
        return _ops().paged_cache_attention(s["q"], s["k_cache"], s["v_cache"], s["table"],
                                            s["lengths"], s["scale"])
    B, H, Hkv, D = c["B"], c["H"], c["Hkv"], c["D"]
    pages = s["table"].long().clamp(min=0)
    k = s["k_cache"][pages].view(B, -1, Hkv, D).float().permute(0, 2, 3, 1)
    q = s["q"].float().view(B, Hkv, H // Hkv, D)
    p = torch.matmul(q, k).mul_(s["scale"])
    del k
    see = torch.arange(p.size(3), device=DEV)[None, :] < s["lengths"][:, None]
    p.masked_fill_(~see[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    v = s["v_cache"][pages].view(B, -1, Hkv, D).float().permute(0, 2, 1, 3)
    o = torch.matmul(p, v).div_(torch.where(total == 0, 1.0, total))
    return o.view(B, H, D).to(s["q"].dtype)


def _append(s):
    kc, vc = s["k_cache"], s["v_cache"]
    if own:
        _ops().paged_cache_append(s["k"], s["v"], s["offsets"], s["starts"], kc, vc, s["table"])
        return kc, vc
    o = s["offsets"].long()
    N, page = s["k"].size(0), kc.size(1)
    b = _list_of_row(o, N)
    at = s["starts"].long()[b] + torch.arange(N, device=DEV) - o[b]
    pages = s["table"].long()[b, at // page]
    kc[pages, at % page] = s["k"]
    vc[pages, at % page] = s["v"]
    return kc, vc


# ---------------------------------------------------------------------------
# Work and the definition in 64 bits
# ---------------------------------------------------------------------------

def _pairs(case: dict, n: np.ndarray) -> int:
    """Visible (query, key) pairs of one head."""
    nk = n + _extras(case, n)
    if not case["causal"]:
        return int((n * nk).sum())
    return int((n * (nk - n) + n * (n + 1) // 2).sum())


def work(case: dict) -> dict:
    n = _lengths(case)
    Hkv, D = case["Hkv"], case["D"]
    if case["kind"] in ("prompt", "train"):
        nq, nk, H = int(n.sum()), int((n + _extras(case, n)).sum()), case["H"]
        pairs = _pairs(case, n)
        if case["kind"] == "prompt":
            return {"bytes": 2 * D * (2 * nq * H + 2 * nk * Hkv), "flops": 4 * D * H * pairs}
        return {"bytes": 2 * D * (4 * nq * H + 4 * nk * Hkv), "flops": 14 * D * H * pairs}
    if case["kind"] == "step":
        return {"bytes": 2 * D * (2 * int(n.sum()) * Hkv + 2 * n.size * case["H"]),
                "flops": 4 * D * case["H"] * int(n.sum())}
    return {"bytes": 2 * D * 4 * int(n.sum()) * Hkv, "flops": 0}


def exact(case: dict, seed: int):
    """The same outputs list by list (and head by head) in 64 bits."""
    s = prepare(case, seed)
    kind = case["kind"]
    with torch.no_grad():
        if kind == "append":
            kc, vc = s["k_cache"].double(), s["v_cache"].double()
            o, starts = s["offsets"].tolist(), s["starts"].tolist()
            page = case["page"]
            for b in range(case["B"]):
                for t0 in range(0, o[b + 1] - o[b]):
                    if t0 and (starts[b] + t0) % page:
                        continue  # inside a page begun before
                    at = starts[b] + t0
                    m = min(page - at % page, o[b + 1] - o[b] - t0)
                    p, r = int(s["table"][b, at // page]), o[b] + t0
                    kc[p, at % page: at % page + m] = s["k"][r: r + m].double()
                    vc[p, at % page: at % page + m] = s["v"][r: r + m].double()
            return kc, vc
        H, Hkv, D = case["H"], case["Hkv"], case["D"]
        G = H // Hkv
        if kind == "step":
            out = torch.zeros((case["B"], H, D), dtype=torch.float64, device=DEV)
            for b, n in enumerate(s["lengths"].tolist()):
                pages = s["table"][b, : -(-n // case["page"])].long()
                k = s["k_cache"][pages].reshape(-1, Hkv, D)[:n].double()
                v = s["v_cache"][pages].reshape(-1, Hkv, D)[:n].double()
                for h in range(Hkv):
                    qh = s["q"][b, h * G:(h + 1) * G].double()
                    w = torch.softmax(qh @ k[:, h].T * s["scale"], dim=-1)
                    out[b, h * G:(h + 1) * G] = w @ v[:, h]
            return out
        q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
        out, dq, dk, dv = (torch.zeros_like(x) for x in (q, q, k, v))
        g = s["grad"].double() if kind == "train" else None
        qo, ko = s["q_offsets"].tolist(), s["k_offsets"].tolist()
        for b in range(case["B"]):
            rq, rk = slice(qo[b], qo[b + 1]), slice(ko[b], ko[b + 1])
            nq, nk = qo[b + 1] - qo[b], ko[b + 1] - ko[b]
            if nq == 0 or nk == 0:
                continue
            hide = None
            if case["causal"]:
                hide = torch.ones((nq, nk), dtype=torch.bool, device=DEV).triu(nk - nq + 1)
            for h in range(H):
                qh, kh, vh = q[rq, h], k[rk, h // G], v[rk, h // G]
                a = qh @ kh.T * s["scale"]
                if hide is not None:
                    a.masked_fill_(hide, -math.inf)
                w = torch.softmax(a, dim=-1)
                out[rq, h] = w @ vh
                if g is not None:
                    gh = g[rq, h]
                    dv[rk, h // G] += w.T @ gh
                    dw = gh @ vh.T
                    da = w * (dw - (w * dw).sum(-1, keepdim=True)) * s["scale"]
                    dq[rq, h] = da @ kh
                    dk[rk, h // G] += da.T @ qh
        return out if kind == "prompt" else (out, dq, dk, dv)

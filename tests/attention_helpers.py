"""Attention over packed lists in float64 (numpy, list by list and head by
head), and how far a correct kernel may be from it.

The bounds are first-order: unit roundoff u of the element type (2^-8 bf16,
2^-11 fp16: round to nearest), 2^-24 of fp32.  A kernel rounds each probability
(or dS) and each result once to the element type; scores, sums and results are
accumulated in fp32, whose worst case for a sum of n terms is n 2^-24 of the
terms' magnitudes.  fp16 values below 2^-14 are subnormal: an absolute 2^-25.
"""

from __future__ import annotations

from dataclasses import dataclass, field

import numpy as np

U = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float16": 2.0 ** -25, "bfloat16": 0.0}
E32 = 2.0 ** -24


@dataclass
class Result:
    out: np.ndarray
    lse: np.ndarray
    out_tol: np.ndarray
    lse_tol: np.ndarray
    dq: np.ndarray | None = None
    dk: np.ndarray | None = None
    dv: np.ndarray | None = None
    dq_tol: np.ndarray = field(default=None)
    dk_tol: np.ndarray = field(default=None)
    dv_tol: np.ndarray = field(default=None)


def visible(nq: int, nk: int, causal: bool) -> np.ndarray:
    see = np.ones((nq, nk), bool)
    if causal:
        see &= np.arange(nk)[None, :] <= np.arange(nq)[:, None] + nk - nq
    return see


def attention(q, k, v, q_offsets, k_offsets, causal, scale, dtype, grad=None) -> Result:
    """q [Nq, H, D], k and v [Nk, Hkv, D], offsets lists; float64 in and out."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    Nq, H, D = q.shape
    Hkv = k.shape[1]
    G = H // Hkv
    u, tiny = U[dtype], TINY[dtype]
    out, out_tol = np.zeros_like(q), np.zeros_like(q)
    lse, lse_tol = np.full((H, Nq), -np.inf), np.zeros((H, Nq))
    r = Result(out, lse, out_tol, lse_tol)
    if grad is not None:
        grad = np.asarray(grad, np.float64)
        r.dq, r.dk, r.dv = np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)
        r.dq_tol, r.dk_tol, r.dv_tol = np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)
    for b in range(len(q_offsets) - 1):
        rq = slice(int(q_offsets[b]), int(q_offsets[b + 1]))
        rk = slice(int(k_offsets[b]), int(k_offsets[b + 1]))
        nq, nk = rq.stop - rq.start, rk.stop - rk.start
        if nq <= 0 or nk <= 0:
            continue
        see = visible(nq, nk, causal)
        some = see.any(1)
        for h in range(H):
            qh, kh, vh = q[rq, h], k[rk, h // G], v[rk, h // G]
            s = np.where(see, qh @ kh.T * scale, -np.inf)
            # Error of a score: D terms summed in fp32, then one product; of
            # its exponential's argument in base 2 with the subtracted maximum
            # or lse, a few roundings of their magnitudes.
            mag = np.abs(qh) @ np.abs(kh).T * scale
            es = float((D + 8) * E32 * mag.max() + 8 * E32)
            top = np.where(some, s.max(1), 0.0)
            e = np.exp(s - top[:, None])
            tot = e.sum(1)
            p = e / np.where(some, tot, 1.0)[:, None]
            o = p @ vh
            ep = 2 * es + (nk / 16 + 16) * E32  # relative, of a normalized probability
            pv = p @ np.abs(vh)
            eo = (u + ep) * pv + tiny * np.abs(vh).sum(0)[None, :]
            out[rq, h] = o
            out_tol[rq, h] = np.where(some[:, None], 1.01 * (eo + u * np.abs(o)) + tiny, 0.0)
            with np.errstate(divide="ignore"):
                lse[h, rq] = np.where(some, top + np.log(tot), -np.inf)
            lse_tol[h, rq] = 2 * es + (nk / 16 + 16) * E32 + 4 * E32 * np.abs(np.where(some, lse[h, rq], 0))
            if grad is None:
                continue
            g = grad[rq, h]
            dp = g @ vh.T
            delta = (g * o).sum(1)
            ds = p * (dp - delta[:, None])
            r.dv[rk, h // G] += p.T @ g
            r.dq[rq, h] = ds @ kh * scale
            r.dk[rk, h // G] += ds.T @ qh * scale
            # delta comes from the rounded output.
            ed = (np.abs(g) * out_tol[rq, h]).sum(1) + (D + 2) * E32 * (np.abs(g) * np.abs(o)).sum(1)
            edp = (D + 2) * E32 * (np.abs(g) @ np.abs(vh).T)
            epg = ep + 4 * E32 * np.abs(np.where(some, lse[h, rq], 0))[:, None]
            eds = np.where(see, p * (edp + ed[:, None]) + (u + epg) * np.abs(ds) + tiny, 0.0)
            epv = np.where(see, p * (u + epg) + tiny, 0.0)
            acc = (max(nq * G, nk) / 16 + 16) * E32
            r.dq_tol[rq, h] += scale * ((eds + acc * np.abs(ds)) @ np.abs(kh))
            r.dk_tol[rk, h // G] += scale * ((eds + acc * np.abs(ds)).T @ np.abs(qh))
            r.dv_tol[rk, h // G] += (epv + acc * p).T @ np.abs(g)
    if grad is not None:
        for x, t in ((r.dq, r.dq_tol), (r.dk, r.dk_tol), (r.dv, r.dv_tol)):
            t += u * (np.abs(x) + t) + tiny
            t *= 1.01
    return r


def paged_attention(q, keys, values, scale, dtype):
    """One query per sequence: q [B, H, D], keys and values a list of [n, Hkv, D]."""
    B, H, D = q.shape
    outs, tols = np.zeros((B, H, D)), np.zeros((B, H, D))
    for b in range(B):
        n = keys[b].shape[0]
        r = attention(q[b:b + 1], keys[b], values[b], [0, 1], [0, n], False, scale, dtype)
        outs[b], tols[b] = r.out[0], r.out_tol[0]
    return outs, tols


def check(got, want, tol, what):
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert np.isfinite(got).all() or not np.isfinite(want).all(), f"{what}: not finite"
    with np.errstate(invalid="ignore"):  # infinities on both sides: equal below
        bad = ~(np.abs(got - want) <= tol)
    bad &= ~((got == want) | (np.isnan(got) & np.isnan(want)))
    if bad.any():
        i = np.unravel_index(np.argmax(np.where(bad, np.abs(got - want) - tol, -np.inf)), got.shape)
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.size} out of tolerance, worst at {i}: "
                             f"{got[i]} vs {want[i]} (tol {tol[i]})")

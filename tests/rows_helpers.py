"""Rotation by position and rows of 4 bits, in plain forms: rotation in fp32 with
every operation rounded by itself (the kernels' own steps) and in float64, 4-bit
rows by the CPU oracle's codec, and attention over them in float64.

Bounds of attention over 4-bit rows, first-order, in the terms of
attention_helpers.  A value is s c + b = s e + f, e = c - 8, |e| <= 8, f = b + 8 s.
The kernel's products sum q (128 + c) - 136 q in fp32, so a score's terms have
magnitudes of up to 144 s |q| + 136 s |q| + |f| |q|; likewise 280 s p for the
second product.  p s is rounded to bf16 (2^-8), for fp16 outputs to two bf16
parts (2^-16); f is rounded to fp32.
"""

from __future__ import annotations

import numpy as np
import torch

import oracle as orc
from attention_helpers import E32, TINY, U

DT = {"float16": torch.float16, "bfloat16": torch.bfloat16}


def make(shape, dtype, seed, scale=1.0):
    x = torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale
    return x.to(DT.get(dtype, dtype))


def angles(positions, R, base=10000.0):
    """[positions, R / 2, 2] cosine and sine in fp32, from 64 bits."""
    w = base ** (-2 * np.arange(R // 2) / R)
    a = np.arange(positions)[:, None] * w
    return torch.from_numpy(np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32))


def positions_of(offsets, starts, N):
    """Each row's list (-1: none) and position."""
    lists, at = np.full(N, -1), np.zeros(N, np.int64)
    for b in range(len(offsets) - 1):
        for r in range(max(0, offsets[b]), min(N, offsets[b + 1])):
            lists[r], at[r] = b, r - offsets[b] + (starts[b] if starts is not None else 0)
    return lists, at


def rotate(x, offsets, table, starts=None, interleaved=False, sign=1, dtype=torch.float32):
    """x [N, H, D] turned, in `dtype` arithmetic (fp32: as the kernels round); rows
    of no list zeros, positions outside the table NaN."""
    N, H, D = x.shape
    lists, at = positions_of(offsets, starts, N)
    y = x.to(dtype).clone()
    y[torch.from_numpy(lists < 0)] = 0
    R = 2 * table.shape[1]
    inside = (lists >= 0) & (at >= 0) & (at < table.shape[0])
    first = np.array([starts[b] if starts is not None and b >= 0 else 0 for b in lists])
    inside &= first >= 0
    outside = torch.from_numpy((lists >= 0) & ~inside)
    y[outside, :, :R] = float("nan")
    rows = torch.from_numpy(np.flatnonzero(inside))
    if rows.numel():
        t = table[torch.from_numpy(at[inside])].to(dtype)
        c, s = t[:, None, :, 0], t[:, None, :, 1] * sign
        xs = x[rows].to(dtype)
        a, b = (xs[..., 0:R:2], xs[..., 1:R:2]) if interleaved else (xs[..., :R // 2], xs[..., R // 2:R])
        u, w = a * c - b * s, b * c + a * s
        turned = torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1)
        y[rows, :, :R] = turned
    return y


def rows4(x):
    """fp32 [..., D] as rows of a 4-bit cache, by the oracle's codec."""
    flat = np.ascontiguousarray(x.float().numpy().reshape(-1, x.shape[-1]))
    q = orc.quantize_fused_nbit(flat, 4)
    return torch.from_numpy(np.ascontiguousarray(q)).reshape(*x.shape[:-1], -1)


def parts4(rows):
    """(scale, bias, codes) of 4-bit rows in float64."""
    r = rows.numpy()
    ends = np.ascontiguousarray(r[..., -4:]).view(np.float16).astype(np.float64)
    c = np.empty((*r.shape[:-1], 2 * (r.shape[-1] - 4)))
    c[..., 0::2], c[..., 1::2] = r[..., :-4] & 15, r[..., :-4] >> 4
    return ends[..., 0], ends[..., 1], c


def values4(rows):
    s, b, c = parts4(rows)
    return c * s[..., None] + b[..., None]


def attention4(q, keys, values, scale, dtype):
    """One query per sequence (q [B, H, D] float64) over lists of 4-bit rows
    [n, Hkv, D / 2 + 4]: float64 outputs and their bounds."""
    B, H, D = q.shape
    out, tol = np.zeros((B, H, D)), np.zeros((B, H, D))
    u, tiny = U[dtype], TINY[dtype]
    up = 2.0 ** -16 if dtype == "float16" else 2.0 ** -8
    for b in range(B):
        n, Hkv = keys[b].shape[:2]
        if n == 0:
            continue
        G = H // Hkv
        ks, kbias, kc = parts4(keys[b])
        vs, vbias, vc = parts4(values[b])
        kf, vf = kbias + 8 * ks, vbias + 8 * vs
        for h in range(H):
            qh, g = q[b, h], h // G
            s = scale * ((kc[:, g] * ks[:, g, None] + kbias[:, g, None]) @ qh)
            mag = scale * np.abs(qh).sum() * (280 * ks[:, g] + np.abs(kf[:, g]))
            es = float((2 * D + 16) * E32 * mag.max() + 8 * E32 * (1 + np.abs(s).max()))
            e = np.exp(s - s.max())
            p = e / e.sum()
            o = p @ (vc[:, g] * vs[:, g, None] + vbias[:, g, None])
            ep = 2 * es + (n / 16 + 16) * E32
            coded = p @ (np.abs(vc[:, g] - 8) * vs[:, g, None])
            flat = p @ np.abs(vf[:, g])
            eo = (up + ep) * coded + (ep + 4 * E32) * flat
            eo = eo + (n / 16 + 16) * E32 * 280 * (p @ vs[:, g])
            out[b, h] = o
            tol[b, h] = 1.01 * (eo + u * np.abs(o)) + tiny
    return out, tol


def page_table(lengths, page, seed=0, extra=3, width=None):
    """Pages in a random order, -1 where a list has none; and their number."""
    rng = np.random.default_rng(seed)
    need = [-(-int(n) // page) for n in lengths]
    order = rng.permutation(sum(need) + extra).astype(np.int32)
    table = np.full((len(lengths), max(need + [1]) if width is None else width), -1, np.int32)
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = order[at: at + m]
        at += m
    return torch.from_numpy(table), order.size

"""How far attention over 4-bit rows may be from its float64 definition on the mean
of the squares: the variances of the kernel's roundings, each uniform over its
step, so of variance step^2 / 12.

A value is s e + f, e = c - 8, f = b + 8 s.  For an output o = sum_j p_j v_j:

* o is rounded to the element type: step^2 / 12 with o's own step;
* p_j s_j is rounded to fp16, a step of at most 2^-10 of it: moves o by that times
  e_j.  (For fp16 outputs a second operand holds what this leaves: a step of 2^-20);
* a score's sums are rounded to fp32 as they run along the head, 32 columns to a
  product: taken as four roundings a product, each of up to 2^-24 of what the sum
  has grown to.  The score itself, its two parts and their difference from the
  maximum: four more.  An error d_j of score j moves o by p_j (v_j - o) d_j;
* sums over tokens run along in fp32, 32 tokens at a time.  Their product takes off
  8 S, S their sum of p s, and adds codes times p s: what stands in it is up to 8 S + R
  where R is what sum p s e has grown to, taken as |sum| + sqrt(sum of squares).  Three
  products (offset, first and second operand), four roundings each: 12.  sum p f, of up
  to A = sum p |f|, in four lanes of eight tokens each: 32 roundings of a quarter of A,
  2 A^2; sum p alike, in parts of o.  Sixteen waves' parts at most are joined.

Independent roundings' variances add up.  An output that is not zero in most of its
tokens has thousands of them behind it, so the mean of error^2 / variance over a few
thousand outputs is near 1 or below, and a token or a weight's bits lost shows.
"""

from __future__ import annotations

import numpy as np

from attention_helpers import E32
from rows_helpers import parts4

# Mantissa bits and the exponent of the smallest normal number.
BITS = {"float16": (10, -14), "bfloat16": (7, -126)}


def step_of(x, dtype):
    """The distance between neighbours of x in the type."""
    bits, least = BITS[dtype]
    e = np.frexp(np.abs(x))[1] - 1
    return 2.0 ** (np.maximum(np.where(x == 0, least, e), least) - bits)


def attention4_errors(q, keys, values, scale, dtype, plant=None):
    """q [B, H, D] float64, lists of 4-bit rows: outputs [B, H, D] and the variances
    of a correct kernel's.  `plant(p)`: weights [n] spoiled before they are summed."""
    B, H, D = q.shape
    out, var = np.zeros((B, H, D)), np.ones((B, H, D))
    ps = 2.0 ** -20 if dtype == "float16" else 2.0 ** -10
    for b in range(B):
        n, Hkv = keys[b].shape[:2]
        if n == 0:
            continue
        G = H // Hkv
        ks, kb, kc = parts4(keys[b])
        vs, vb, vc = parts4(values[b])
        for h in range(H):
            qh, g = q[b, h], h // G
            s = scale * ((kc[:, g] * ks[:, g, None] + kb[:, g, None]) @ qh)
            # What the sum over columns has grown to, behind every 32 of them.
            run = np.abs(np.cumsum(kc[:, g] * qh, -1) - 8 * qh.sum())[:, 31 if D > 31 else D - 1::32]
            first = np.abs(8 * qh.sum()) + np.abs(qh).sum()
            sums = (run ** 2 * 4).sum(-1) + 4 * first ** 2
            sd2 = E32 ** 2 * ((scale * ks[:, g]) ** 2 * sums
                              + 4 * (s ** 2 + (scale * (kb[:, g] + 8 * ks[:, g]) * qh.sum()) ** 2 + s.max() ** 2 + 1))
            e = np.exp(s - s.max())
            p = e / e.sum()
            w = plant(p.copy()) if plant is not None else p
            v = vc[:, g] * vs[:, g, None] + vb[:, g, None]
            o = w @ v
            pse = (p * vs[:, g])[:, None] * (vc[:, g] - 8)
            grown = np.abs(pse.sum(0)) + np.sqrt((pse ** 2).sum(0))
            flat = p @ np.abs(vb[:, g] + 8 * vs[:, g])
            tiles = np.add.reduceat(p * vs[:, g], np.arange(0, n, 32))
            runs = E32 ** 2 * (12 * ((8 * tiles[:, None] + grown) ** 2).sum(0)
                               + len(tiles) * 2 * (flat ** 2 + o ** 2) + 16 * (flat + grown) ** 2)
            out[b, h] = o
            var[b, h] = (step_of(o, dtype) ** 2 / 12
                         + ps ** 2 / 12 * (pse ** 2).sum(0) + runs
                         + ((p[:, None] * (v - o)) ** 2 * sd2[:, None]).sum(0))
    return out, var


def mean_square(got, want, var):
    """The mean of error^2 / variance: about 1 at most."""
    return float((((got - want) ** 2) / var).mean())

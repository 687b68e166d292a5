"""The mean-square bound of attention over 4-bit rows sees lost work: mistakes are
planted in the weights of its definition, on the CPU."""

import numpy as np
import pytest
import torch

from int4_errors import attention4_errors, mean_square, step_of
from rows_helpers import make, rows4

LIMIT = 1.3  # of the mean square over 4,096 outputs or more (their own spread: 2 percent)


def half_steps(x, bits):
    """Rounded to `bits` mantissa bits."""
    e = 2.0 ** (np.frexp(x)[1] - 1 - bits)
    return np.where(x == 0, 0, np.rint(x / np.where(x == 0, 1, e)) * e)


def lose(first, count):
    def plant(p):
        p[first:first + count] = 0
        return p / p.sum()
    return plant


def case(n, D, H, dtype):
    q = make((1, H, D), dtype, n + D).double().numpy()
    return q, [rows4(make((n, 1, D), torch.float32, 1))], [rows4(make((n, 1, D), torch.float32, 2))]


def rounded(x, dtype):
    return torch.from_numpy(x).to(getattr(torch, dtype)).double().numpy()


def test_steps():
    assert step_of(np.array([1.0, 1.5, 2.0, 0.0, 2.0 ** -20]), "float16").tolist() == [
        2.0 ** -10, 2.0 ** -10, 2.0 ** -9, 2.0 ** -24, 2.0 ** -24]
    assert step_of(np.array([1.0, -3.0]), "bfloat16").tolist() == [2.0 ** -7, 2.0 ** -6]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("n,D", [(200, 128), (1000, 64), (5000, 64), (3000, 128)])
def test_what_it_sees(dtype, n, D):
    q, k, v = case(n, D, 4096 // D, dtype)
    want, var = attention4_errors(q, k, v, D ** -0.5, dtype)
    assert mean_square(rounded(want, dtype), want, var) <= 1.05
    # Weights with the kernel's own bits pass, with fewer they do not.
    bits = 10 if dtype == "bfloat16" else 21
    ok, _ = attention4_errors(q, k, v, D ** -0.5, dtype, lambda p: half_steps(p, bits))
    assert mean_square(rounded(ok, dtype), want, var) <= LIMIT
    for plant in (lose(n // 3, 1) if n <= 1000 else lose(n // 3, 8), lose(64, 32), lose(128, 128), lose(n - 32, 32),
                  lambda p: half_steps(p, 4), lambda p: half_steps(p, 7 if dtype == "bfloat16" else 10)):
        bad, _ = attention4_errors(q, k, v, D ** -0.5, dtype, plant)
        assert mean_square(rounded(bad, dtype), want, var) > LIMIT


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("mean", [0.0, 1.0])
def test_score_errors_of_half_a_thousandth_show_in_fp16(D, mean):
    """What sums that stand on 1024 times the queries' sum lose (4e-4 and more of a
    score, for queries of mean 1)."""
    q, k, v = case(400, D, 4096 // D, "float16")
    q = q + mean
    want, var = attention4_errors(q, k, v, D ** -0.5, "float16")
    rng = np.random.default_rng(0)
    bad, _ = attention4_errors(q, k, v, D ** -0.5, "float16",
                               lambda p: (lambda w: w / w.sum())(p * np.exp(rng.normal(0, 4e-4, p.size))))
    assert mean_square(rounded(bad, "float16"), want, var) > LIMIT

"""Attention cut over blocks in ways that meet only at some sizes: heads packed into
blocks whose keys two groups of waves share, and tiles found by rank or planned
beforehand at every padded head width.  Against the float64 definition."""

import numpy as np
import pytest

from test_gpu_attention import make, offsets_of, run

pytestmark = pytest.mark.gpu


def inputs(qo, ko, H, Hkv, D, dtype, more=0):
    Nq, Nk = int(qo[-1]) + more, int(ko[-1]) + more
    return (make(Nq, H, D, dtype, 1), make(Nk, Hkv, D, dtype, 2), make(Nk, Hkv, D, dtype, 3),
            make(Nq, H, D, dtype, 4))


@pytest.mark.parametrize("H,Hkv", [(8, 2), (6, 3), (4, 1)])
@pytest.mark.parametrize("D,dtype", [(24, "float16"), (64, "bfloat16"), (96, "float16"), (128, "bfloat16")])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_heads_over_two_groups_of_keys(dev, H, Hkv, D, dtype, causal):
    """Few short query lists behind long ones of keys (512 or more on average), with
    shared heads: four or two heads of a block, and its keys over two groups."""
    qo = offsets_of([100, 0, 1, 33, 128, 129]) + 3
    ko = offsets_of([900, 700, 1500, 5, 0, 1200]) + 2
    q, k, v, g = inputs(qo, ko, H, Hkv, D, dtype, 4)
    run(dev, q, k, v, qo, ko, causal, None, dtype, g)


@pytest.mark.parametrize("Hkv", [16, 32, 64])
@pytest.mark.parametrize("D,dtype", [(64, "float16"), (96, "bfloat16"), (128, "float16")])
def test_ranked_tiles(dev, Hkv, D, dtype):
    """Up to 62 lists of 512 rows or more on average, more tiles than start at once."""
    qo, ko = offsets_of([400, 1, 330, 410]), offsets_of([900, 1300, 300, 1200])
    q, k, v, g = inputs(qo, ko, 64, Hkv, D, dtype)
    run(dev, q, k, v, qo, ko, True, None, dtype, g)


@pytest.mark.parametrize("Hkv", [16, 64])
@pytest.mark.parametrize("D,dtype", [(64, "bfloat16"), (96, "float16"), (128, "bfloat16")])
def test_planned_tiles(dev, Hkv, D, dtype):
    """Too many lists to rank and enough tiles (4096) for an order worked out beforehand,
    in both directions."""
    rng = np.random.default_rng(Hkv + D)
    nq, nk = rng.integers(0, 271, 64), rng.integers(0, 271, 64)
    nq[7], nk[7], nq[20], nk[30] = 600, 300, 0, 0
    qo, ko = offsets_of(nq), offsets_of(nk) + 1
    q, k, v, g = inputs(qo, ko, 64, Hkv, D, dtype, 200)
    assert -(-q.size(0) // 128) * 64 > 4096
    run(dev, q, k, v, qo, ko, True, None, dtype, g)

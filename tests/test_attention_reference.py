"""The float64 attention the GPU tests compare with, checked on the CPU: against
torch's softmax and autograd, and its gradients against differences."""

import numpy as np
import pytest
import torch

from attention_helpers import attention, visible


def _inputs(nq, nk, H, Hkv, D, seed=0):
    rng = np.random.default_rng(seed)
    return (rng.standard_normal((nq, H, D)), rng.standard_normal((nk, Hkv, D)),
            rng.standard_normal((nk, Hkv, D)), rng.standard_normal((nq, H, D)))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("qo,ko", [([0, 3, 3, 8], [0, 3, 3, 8]), ([0, 4, 6], [0, 9, 10])])
def test_against_torch(qo, ko, causal):
    q, k, v, g = _inputs(qo[-1], ko[-1], 4, 2, 8)
    r = attention(q, k, v, qo, ko, causal, 0.3, "bfloat16", g)
    tq, tk, tv = (torch.tensor(x, requires_grad=True) for x in (q, k, v))
    rows = []
    for b in range(len(qo) - 1):
        a, c = tq[qo[b]:qo[b + 1]].transpose(0, 1), tk[ko[b]:ko[b + 1]].transpose(0, 1)
        see = torch.from_numpy(visible(a.size(1), c.size(1), causal))
        w = torch.softmax((a @ c.repeat_interleave(2, 0).transpose(1, 2) * 0.3).masked_fill(~see, -np.inf), -1)
        w = torch.nan_to_num(w)  # rows that see nothing
        rows.append((w @ tv[ko[b]:ko[b + 1]].transpose(0, 1).repeat_interleave(2, 0)).transpose(0, 1))
    out = torch.cat(rows)
    np.testing.assert_allclose(r.out, out.detach().numpy(), atol=1e-12)
    if all((qo[b + 1] - qo[b]) <= (ko[b + 1] - ko[b]) for b in range(len(qo) - 1)):
        dq, dk, dv = torch.autograd.grad(out, (tq, tk, tv), torch.from_numpy(g))
        for x, y in ((r.dq, dq), (r.dk, dk), (r.dv, dv)):
            np.testing.assert_allclose(x, y.numpy(), atol=1e-12)


@pytest.mark.parametrize("qo,ko", [([0, 5], [0, 5]), ([0, 6], [0, 3]), ([0, 2, 4], [0, 7, 9])])
def test_gradients_against_differences(qo, ko):
    q, k, v, g = _inputs(qo[-1], ko[-1], 2, 1, 8, seed=3)
    r = attention(q, k, v, qo, ko, True, 0.4, "bfloat16", g)
    rng = np.random.default_rng(7)
    for i, grad in enumerate((r.dq, r.dk, r.dv)):
        step = rng.standard_normal(grad.shape)
        def loss(t):
            x = [q, k, v]
            x[i] = x[i] + t * step
            return float((attention(*x, qo, ko, True, 0.4, "bfloat16").out * g).sum())
        diff = (loss(1e-5) - loss(-1e-5)) / 2e-5
        assert abs(diff - float((grad * step).sum())) < 1e-7 * (1 + abs(diff))


def test_a_query_that_sees_nothing_is_zero():
    q, k, v, g = _inputs(5, 2, 1, 1, 8)
    r = attention(q, k, v, [0, 5], [0, 2], True, 1.0, "float16", g)
    assert (r.out[:3] == 0).all() and np.isneginf(r.lse[0, :3]).all() and (r.dq[:3] == 0).all()
    assert (r.out[3:] != 0).all()

"""Derivatives that jagged_attention does not have are refused, wherever its tensors are
(no GPU needed: the refusal comes first)."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

import mx_fbgemm  # noqa: F401


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("requires_grad", [False, True])
def test_tangents_are_refused(which, requires_grad):
    x = [torch.zeros((4, 2, 32), dtype=torch.float16) for _ in range(3)]
    o = torch.tensor([0, 4])
    with fwad.dual_level():
        x[which] = fwad.make_dual(x[which], torch.ones_like(x[which]))
        x[0 if which else 1].requires_grad_(requires_grad)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.ops.mx_fbgemm.jagged_attention(*x, o)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            torch.ops.mx_fbgemm.jagged_attention(*x, o)
        # With forward mode switched off, and without tangents, it is the device that is wrong.
        with fwad._set_fwd_grad_enabled(False), pytest.raises((RuntimeError, NotImplementedError)) as e:
            torch.ops.mx_fbgemm.jagged_attention(*x, o)
        assert "forward-mode" not in str(e.value)
    with pytest.raises((RuntimeError, NotImplementedError)) as e:
        torch.ops.mx_fbgemm.jagged_attention(*(t.detach() for t in x), o)
    assert "forward-mode" not in str(e.value)

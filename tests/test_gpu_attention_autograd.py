"""What autograd is told about the attention operators."""

import pytest
import torch

pytestmark = pytest.mark.gpu

OPS = torch.ops.mx_fbgemm


def cache_args(dev):
    kc, vc = (torch.ones((4, 4, 2, 32), dtype=torch.bfloat16, device=dev) for _ in range(2))
    k, v = (torch.full((3, 2, 32), 2.0, dtype=torch.bfloat16, device=dev) for _ in range(2))
    table = torch.tensor([[1, 3]], dtype=torch.int32, device=dev)
    return k, v, torch.tensor([0, 3], device=dev), torch.tensor([2], device=dev), kc, vc, table


def test_an_append_is_an_in_place_change(dev):
    """The caches' versions count appends: a backward that has saved one notices."""
    args = cache_args(dev)
    kc, vc = args[4:6]
    before = kc._version, vc._version
    OPS.paged_cache_append(*args)
    assert (kc._version, vc._version) == (before[0] + 1, before[1] + 1)
    for which in (kc, vc):
        w = torch.ones(32, device=dev, dtype=torch.bfloat16, requires_grad=True)
        y = (which * w).sum()
        OPS.paged_cache_append(*args)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    (kc * w).sum().backward()
    assert torch.isfinite(w.grad).all()


def test_a_view_shares_its_caches_version(dev):
    both = torch.ones((4, 2, 4, 2, 32), dtype=torch.bfloat16, device=dev)
    k, v, off, starts, _, _, table = cache_args(dev)
    before = both._version
    OPS.paged_cache_append(k, v, off, starts, both[:, 0], both[:, 1], table)
    assert both._version == before + 2 and float(both[1, 0, 2, 0, 0]) == 2.0


def test_appends_without_versions(dev):
    """A refused append changes none; caches made in inference mode have none."""
    args = cache_args(dev)
    kc = args[4]
    before = kc._version
    with pytest.raises(RuntimeError):
        OPS.paged_cache_append(args[0], args[1][:2], *args[2:])
    assert kc._version == before
    with torch.inference_mode():
        inner = cache_args(dev)
        OPS.paged_cache_append(*inner)
        OPS.paged_cache_append(*args)
    OPS.paged_cache_append(*inner)                                  # outside it
    OPS.paged_cache_append(*args[:4], *inner[4:6], args[6])         # among ordinary ones
    for c in (*inner[4:6], *args[4:6]):
        assert float(c[1, 2, 0, 0]) == 2.0 and float(c[1, 1, 0, 0]) == 1.0 and float(c[3, 0, 0, 0]) == 2.0

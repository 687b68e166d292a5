"""No gradient flows through the caches: the calls that would cut one refuse."""

import pytest
import torch

from rows_helpers import angles, make

pytestmark = pytest.mark.gpu

OPS = torch.ops.mx_fbgemm


def setup(dev, four):
    kind = torch.uint8 if four else torch.float16
    kc, vc = (torch.zeros((2, 4, 1, 12 if four else 16), dtype=kind, device=dev) for _ in range(2))
    x = make((1, 1, 16), "float16", 1).to(dev)
    off, starts = torch.tensor([0, 1], device=dev), torch.tensor([0], device=dev)
    return dict(q=x, k=x.clone(), v=x.clone(), offsets=off, starts=starts, table=angles(4, 16).to(dev), k_cache=kc,
                v_cache=vc, page_table=torch.tensor([[1]], dtype=torch.int32, device=dev))


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("name", ["q", "k", "v", "table"])
def test_rotating_append(dev, four, name):
    a = setup(dev, four)
    plain = a[name]
    a[name] = plain.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        OPS.paged_cache_append_rotary(**a)
    assert torch.count_nonzero(a["k_cache"]) == 0 and a["k_cache"]._version == 0
    with torch.no_grad():
        got = OPS.paged_cache_append_rotary(**a)
    assert torch.equal(got, OPS.paged_cache_append_rotary(**{**a, name: plain}))
    with torch.autograd.forward_ad.dual_level():
        a[name] = torch.autograd.forward_ad.make_dual(plain, torch.ones_like(plain))
        with pytest.raises(NotImplementedError, match="forward"):
            OPS.paged_cache_append_rotary(**a)


@pytest.mark.parametrize("name", ["k_cache", "v_cache"])
def test_reading_back(dev, name):
    a = setup(dev, False)
    args = dict(k_cache=a["k_cache"], v_cache=a["v_cache"], page_table=a["page_table"], offsets=a["offsets"], total=1)
    plain = args[name]
    args[name] = plain.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        OPS.paged_cache_gather(**args)
    with torch.no_grad():
        OPS.paged_cache_gather(**args)
    with torch.autograd.forward_ad.dual_level():
        args[name] = torch.autograd.forward_ad.make_dual(plain, torch.ones_like(plain))
        with pytest.raises(NotImplementedError, match="forward"):
            OPS.paged_cache_gather(**args)
    with torch.inference_mode():
        args[name] = plain
        k, v = OPS.paged_cache_gather(**args)
    assert k.shape == (1, 1, 16) and not k.requires_grad

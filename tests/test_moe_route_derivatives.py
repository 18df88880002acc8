"""What the ways to the experts and back do with derivatives that they do not have."""

import pytest
import torch
from torch.autograd import forward_ad

from tilegym_amd import _lib, ops

from .test_int8_ops import gen, routing


def _order(tokens, k):
    rows = torch.arange(tokens * k, dtype=torch.int32).view(tokens, k)
    return ops.MoeOrder(torch.tensor([0, tokens * k], dtype=torch.int32), rows, rows.flatten())


def _refusals(order, x, y, w, dual):
    t = torch.ops.tilegym_hip
    calls = [lambda: ops.moe_permute(dual(x), order), lambda: ops.moe_unpermute(dual(y), order), lambda: ops.moe_unpermute(dual(y), order, w),
             lambda: ops.moe_unpermute(y, order, dual(w))]
    if x.is_cuda:
        calls += [lambda: t.moe_permute(dual(x), order.rows), lambda: t.moe_unpermute(y, order.rows, dual(w))]
    for call in calls:
        with pytest.raises(NotImplementedError):
            call()


def test_forward_mode_is_refused():
    """Not a value without its tangent; in front of everything else that is looked at."""
    x, y, w = torch.zeros(3, 8), torch.zeros(6, 8), torch.ones(3, 2)
    with forward_ad.dual_level():
        for leaf in (False, True):
            _refusals(_order(3, 2), x, y, w, lambda v: forward_ad.make_dual(v.clone().requires_grad_(leaf), torch.ones_like(v)))
            with torch.no_grad(), pytest.raises(NotImplementedError):
                ops.moe_permute(forward_ad.make_dual(x, torch.ones_like(x)), _order(3, 2))
        for call in (lambda: ops.moe_permute(x, _order(3, 2)), lambda: ops.moe_unpermute(y, _order(3, 2), w)):
            with pytest.raises(RuntimeError, match="HIP device"):  # (tensors without a tangent go on to the check of their device)
                call()


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_forward_mode_is_refused_on_a_device(device, monkeypatch, native):
    if not native:
        monkeypatch.setattr(_lib, "native_path", lambda: False)
    order = ops.moe_sort(routing(5, 4, 2, 1).to(device), 4)
    x, y, w = (torch.randn(*s, generator=gen(i)).to(device) for i, s in enumerate(((5, 64), (10, 64), (5, 2))))
    with forward_ad.dual_level():
        for leaf in (False, True):
            _refusals(order, x, y, w, lambda v: forward_ad.make_dual(v.clone().requires_grad_(leaf), torch.ones_like(v)))
        assert torch.equal(ops.moe_unpermute(ops.moe_permute(x, order), order), 2 * x)
    with pytest.raises(NotImplementedError):
        torch.func.jvp(lambda v: ops.moe_permute(v, order), (x,), (x,))

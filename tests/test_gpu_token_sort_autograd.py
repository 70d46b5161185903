"""Derivatives that the token sort does not have are errors, not lost."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


def sorted_case(dev):
    import mtp_b200
    x = torch.randn(6, 8, device=dev)
    ids = torch.randint(0, 3, (6, 2), device=dev, dtype=torch.int32)
    return x, ids, mtp_b200.sort_tokens(x, ids, 3), torch.rand(6, 2, device=dev)


@pytest.mark.parametrize("grad_enabled", [True, False])
def test_forward_mode_raises(cuda_device, grad_enabled):
    import mtp_b200
    x, ids, r, w = sorted_case(cuda_device)
    dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_enabled):
        for call in (lambda: mtp_b200.sort_tokens(dual(x), ids, 3),
                     lambda: mtp_b200.unsort_tokens(dual(r.rows), r.positions, w),
                     lambda: mtp_b200.unsort_tokens(dual(r.rows), r.positions),
                     lambda: mtp_b200.unsort_tokens(r.rows, r.positions, dual(w))):
            with pytest.raises(RuntimeError, match="jvp|forward mode"):
                call()
        # plain tensors pass inside a level
        assert torch.equal(mtp_b200.sort_tokens(x, ids, 3).rows, r.rows)


def test_no_grad_records_nothing(cuda_device):
    import mtp_b200
    x, ids, r, w = sorted_case(cuda_device)
    with torch.no_grad():
        assert not mtp_b200.sort_tokens(x.requires_grad_(), ids, 3).rows.requires_grad
        assert not mtp_b200.unsort_tokens(r.rows, r.positions, w.requires_grad_()).requires_grad

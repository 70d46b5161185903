"""A row of a layer norm is good or bad as a whole. A thread whose wait for its row ran out adds NaN to its part of the
row's sums, as a NaN among its values does: wherever in the row that is, all of the row has to be NaN and no other."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("h", [16, 48, 257, 512, 1001, 2048, 4100, 8192, 9000, 16384])
def test_one_nan_anywhere(cuda_device, dtype, h):
    """Every third row has one NaN, whose column steps through the row: all lanes, warps and vectors, and both rows of a
    pair that shares a barrier."""
    import mtp_b200
    m = 1200
    g = torch.Generator(device="cuda").manual_seed(h)
    x = torch.randn(m, h, generator=g, device="cuda").to(dtype)
    w, b = (torch.randn(h, generator=g, device="cuda") for _ in range(2))
    gy = torch.randn(m, h, generator=g, device="cuda").to(dtype)

    def results(x):
        x = x.detach().requires_grad_()
        y = mtp_b200.layer_norm(x, w, b)
        return y.detach(), torch.autograd.grad(y, x, gy)[0]

    clean = results(x)
    bad = torch.arange(0, m, 3, device="cuda")
    dirty = x.clone()
    dirty[bad, (bad // 3 * 37) % h] = float("nan")
    good = torch.ones(m, dtype=torch.bool, device="cuda")
    good[bad] = False
    for got, want in zip(results(dirty), clean):
        assert torch.isnan(got[bad]).all()
        assert torch.equal(got[good], want[good]) and torch.isfinite(got[good]).all()

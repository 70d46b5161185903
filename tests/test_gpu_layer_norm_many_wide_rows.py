"""Rows wider than the ring kernels take, more of them than the plain kernels have CTAs (32768)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,h", [(torch.bfloat16, 16385), (torch.float32, 11300)])
def test_rows_behind_the_last_cta(cuda_device, dtype, h):
    """Each row is as in a call of its own with its neighbours; the sums over the rows add those of the parts."""
    import mtp_b200
    m, part = 33001, 11001
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(m, h, generator=g, device="cuda", dtype=dtype)
    gy = torch.randn(m, h, generator=g, device="cuda", dtype=dtype)
    w, b = (torch.randn(h, generator=g, device="cuda") for _ in range(2))

    def results(rows):
        leaves = [t.detach().requires_grad_() for t in (x[rows], w, b)]
        y = mtp_b200.layer_norm(*leaves)
        return y.detach(), *torch.autograd.grad(y, leaves, gy[rows])

    y, dx, dw, db = results(slice(None))
    sums = [torch.zeros(h, device="cuda", dtype=torch.float64) for _ in range(2)]
    for start in range(0, m, part):
        rows = slice(start, min(start + part, m))
        py, pdx, pdw, pdb = results(rows)
        assert torch.equal(y[rows], py) and torch.equal(dx[rows], pdx)
        sums[0] += pdw.double()
        sums[1] += pdb.double()
    # 64 parts of at most m / 64 + 1 rows, then 8 and 8 additions: (m / 64 + 20) u of the terms' absolute values on either
    # side. |g xhat| and |g| of normal values have means below 0.7 and 0.8; 1 is more than 40 deviations of their means above.
    bound = 2 * (m / 64 + 20) * 2.0 ** -24 * m
    for got, want in zip((dw, db), sums):
        assert ((got.double() - want).abs() <= bound).all()

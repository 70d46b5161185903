"""Layer norm and its gradients against the definition in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, HALF, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24


def half_step(t):
    """Half a step of rounding to t, relative to the value, and below the smallest normal one."""
    i = torch.finfo(t)
    return i.eps / 2, i.smallest_normal * i.eps / 2


def check(x, w, b, eps=1e-5, grad=None):
    import mtp_b200
    m, h = x.numel() // x.shape[-1], x.shape[-1]
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, w, b)]
    y = mtp_b200.layer_norm(*leaves, eps)
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
    g = torch.randn(x.shape, device=x.device).to(x.dtype) if grad is None else grad
    got = torch.autograd.grad(y, [t for t in leaves if t is not None], g)

    x64, g64 = x.detach().double().reshape(m, h), g.double().reshape(m, h)
    w64 = torch.ones(h, device=x.device, dtype=torch.float64) if w is None else w.detach().double()
    b64 = torch.zeros(h, device=x.device, dtype=torch.float64) if b is None else b.detach().double()
    mean = x64.mean(-1, keepdim=True)
    rstd = 1 / (x64.var(-1, unbiased=False, keepdim=True) + eps).sqrt()
    xhat = (x64 - mean) * rstd
    exact = xhat * w64 + b64
    wg = g64 * w64
    s1, s2 = wg.mean(-1, keepdim=True), (wg * xhat).mean(-1, keepdim=True)

    # No chain of additions in a row's sums is longer than d: each lane adds up at most h / 32 values, then 5 steps
    # of a warp and 32 warps. A relative error of d u of the sum of absolute values each.
    d = h / 32 + 40
    dxhat = U * (d * rstd * x64.abs().mean(-1, keepdim=True) + (d + 8) * xhat.abs())
    rel, tiny = half_step(x.dtype)
    bound = w64.abs() * dxhat + 3 * U * ((w64 * xhat).abs() + b64.abs()) + rel * exact.abs() + tiny
    error = (y.detach().double().reshape(m, h) - exact).abs()
    assert (error <= bound * (1 + 2 * rel)).all(), float((error / bound).max())

    dx = rstd * (wg - s1 - xhat * s2)
    spread = (wg.abs() * dxhat).mean(-1, keepdim=True)
    bound = rstd * ((d + 8) * U * (wg.abs() + wg.abs().mean(-1, keepdim=True) + xhat.abs() * (wg * xhat).abs().mean(-1, keepdim=True))
                    + s2.abs() * dxhat + xhat.abs() * spread)
    bound = bound + (d + 8) * U * dx.abs() + rel * dx.abs() + tiny
    error = (got[0].double().reshape(m, h) - dx).abs()
    assert got[0].shape == x.shape and got[0].dtype == x.dtype
    assert (error <= bound * (1 + 2 * rel)).all(), float((error / bound).max())

    # a column's sum: a chain of at most m / 32 + 64 additions
    chain, at = (m / 32 + 64) * U, 1
    for t, terms, inner in ((w, g64 * xhat, g64.abs() * dxhat), (b, g64, torch.zeros_like(g64))):
        if t is None:
            continue
        rel, tiny = half_step(t.dtype)
        want = terms.sum(0)
        bound = chain * terms.abs().sum(0) + inner.sum(0) + rel * want.abs() + tiny
        error = (got[at].double() - want).abs()
        assert got[at].dtype == t.dtype
        assert (error <= bound * (1 + 2 * rel)).all(), float((error / bound).max())
        at += 1


def inputs(m, h, dtype, params, seed=0, affine=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(m, h, generator=g, device="cuda") * (1 + 7 * (torch.rand(h, generator=g, device="cuda") < 0.05))
    x = (x + 0.5 * torch.randn(m, 1, generator=g, device="cuda")).to(dtype)
    if not affine:
        return x, None, None
    return x, (1 + 0.2 * torch.randn(h, generator=g, device="cuda")).to(params), (0.2 * torch.randn(h, generator=g, device="cuda")).to(params)


SIZES = [(1, 1), (1, 2048), (2, 3), (3, 8), (5, 17), (4, 31), (33, 64), (7, 100), (9, 250), (300, 257), (64, 512), (65, 1000),
         (40, 1001), (17, 1024), (129, 2047), (130, 2048), (20, 4096), (6, 5000), (3, 8192), (3, 8191), (2, 16384), (2, 20001),
         (2, 40000), (5000, 96), (3000, 16)]


@pytest.mark.parametrize("m,h", SIZES)
@pytest.mark.parametrize("dtype", [BF, HALF, F32])
def test_sizes(cuda_device, m, h, dtype):
    check(*inputs(m, h, dtype, F32))


@pytest.mark.parametrize("m,h", [(1, 64), (200, 2048), (33, 999), (2, 70000), (1200, 24)])
@pytest.mark.parametrize("dtype", [BF, HALF])
def test_parameters_of_the_rows_type(cuda_device, m, h, dtype):
    check(*inputs(m, h, dtype, dtype))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("h", [96, 1537, 2048])
def test_without_weight_or_bias(cuda_device, dtype, h):
    x, w, b = inputs(50, h, dtype, F32)
    check(x, None, None)
    check(x, w, None)
    check(x, None, b)


def test_other_dimensions(cuda_device):
    x, w, b = inputs(24, 64, F32, F32)
    check(x.view(2, 3, 4, 64), w, b)
    check(x[0], w, b)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("h,offset,wide", [(2048, 8, 2064), (2048, 1, 2051), (777, 3, 800), (64, 0, 65), (128, 2, 130)])
def test_rows_of_a_wider_tensor(cuda_device, dtype, h, offset, wide):
    x, _, _ = inputs(70, wide, dtype, F32)
    _, w, b = inputs(1, h, dtype, F32)
    check(x[:, offset:offset + h], w, b)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_starts_off_16_bytes(cuda_device, dtype):
    """Every tensor begins inside a 16-byte unit."""
    import mtp_b200
    x, w, b = inputs(30, 256, dtype, dtype)
    shifted = []
    for t in (x, w, b):
        buf = torch.empty(t.numel() + 1, dtype=dtype, device="cuda")
        buf[1:] = t.flatten()
        shifted.append(buf[1:].view(t.shape))
    check(*shifted)


def test_offsets_cost_no_digits(cuda_device):
    """Rows of a large mean and a small spread: the variance comes from centred values."""
    import mtp_b200
    for h in (64, 1024, 2048, 33000):
        x = (4096 + torch.arange(h, device="cuda") % 2).float()[None].repeat(3, 1)  # 4096 and 4097, exact in the sums
        y = mtp_b200.layer_norm(x, eps=0.0)
        # the mean 4096.5 is a number of fp32; a sum's rounding moves it by at most (h / 32 + 40) u 4096.5, against a spread of 0.5
        d = (h / 32 + 40) * U * 4096.5
        assert ((y.abs() - 1).abs() <= 4 * d + 16 * U).all()


@pytest.mark.parametrize("h", [32, 2048, 3001])
def test_constant_rows(cuda_device, h):
    import mtp_b200
    x, w, b = inputs(4, h, F32, F32)
    x[1] = 2.0
    x[2] = 0.0
    y = mtp_b200.layer_norm(x, w, b)
    assert torch.equal(y[1], b) and torch.equal(y[2], b)
    x.requires_grad_()
    y = mtp_b200.layer_norm(x, w, b)
    (grad,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.isfinite(grad).all()
    with torch.no_grad():
        assert torch.isnan(mtp_b200.layer_norm(x, w, b, 0.0)[1:3]).all()  # 0 / 0, as the formula has it


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("h", [48, 2048])
def test_bad_values_stay_in_their_row(cuda_device, bad, h):
    import mtp_b200
    x, w, b = inputs(9, h, F32, F32)
    clean = mtp_b200.layer_norm(x, w, b)
    x[4, 7] = bad
    y = mtp_b200.layer_norm(x, w, b)
    assert torch.isnan(y[4]).all()
    rest = [0, 1, 2, 3, 5, 6, 7, 8]
    assert torch.equal(y[rest], clean[rest])
    x.requires_grad_()
    w.requires_grad_()
    dx, dw = torch.autograd.grad(mtp_b200.layer_norm(x, w, b), (x, w), torch.ones_like(x))
    assert torch.isnan(dx[4]).all() and torch.isfinite(dx[rest]).all() and torch.isnan(dw).all()


def test_no_rows(cuda_device):
    import mtp_b200
    x = torch.zeros(0, 40, device="cuda", requires_grad=True)
    w = torch.ones(40, device="cuda", requires_grad=True)
    b = torch.ones(40, device="cuda", requires_grad=True)
    y = mtp_b200.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y.sum(), (x, w, b))
    assert y.shape == (0, 40) and dx.shape == (0, 40) and not dw.any() and not db.any()


def test_only_the_gradients_asked_for(cuda_device):
    import mtp_b200
    x, w, b = inputs(100, 512, BF, F32)
    g = torch.randn(100, 512, device="cuda").to(BF)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    whole = torch.autograd.grad(mtp_b200.layer_norm(*leaves), leaves, g)
    for i in range(3):
        some = [t.detach().requires_grad_(i == j) for j, t in enumerate(leaves)]
        (got,) = torch.autograd.grad(mtp_b200.layer_norm(*some), [some[i]], g)
        assert torch.equal(got, whole[i])


def test_gradient_against_differences(cuda_device):
    import mtp_b200
    x, w, b = inputs(12, 80, F32, F32)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    g = torch.randn(12, 80, device="cuda")
    grads = torch.autograd.grad(mtp_b200.layer_norm(*leaves), leaves, g)

    def loss(x, w, b):
        y = (x - x.mean(-1, keepdim=True)) / (x.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt() * w + b
        return (y * g).sum()

    at = [t.detach().double() for t in leaves]
    for i in range(3):
        d = torch.randn(at[i].shape, device="cuda", dtype=torch.float64)
        h = 1e-5
        step = lambda s: loss(*(t + s * d if i == j else t for j, t in enumerate(at)))
        slope = (step(h) - step(-h)) / (2 * h)
        # h^2 of the third derivative, and the gradient's own 2^-17
        assert abs(float((grads[i].double() * d).sum() - slope)) <= 2.0 ** -17 * float((grads[i].double() * d).abs().sum()) + 1e-6


def test_same_bits_again(cuda_device):
    import mtp_b200
    x, w, b = inputs(3000, 2048, BF, F32)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    g = torch.randn(3000, 2048, device="cuda").to(BF)
    first = torch.autograd.grad(mtp_b200.layer_norm(*leaves), leaves, g)
    for _ in range(3):
        for p, q in zip(torch.autograd.grad(mtp_b200.layer_norm(*leaves), leaves, g), first):
            assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m,h,wide", [(6000, 1, 3), (5000, 8, 24), (4000, 24, 25), (3000, 40, 64), (700, 5000, 5001), (500, 8200, 8208)])
def test_many_rows_of_a_wider_tensor(cuda_device, dtype, m, h, wide):
    x, _, _ = inputs(m, wide, dtype, F32)
    _, w, b = inputs(1, h, dtype, F32)
    check(x[:, wide - h:], w, b)


@pytest.mark.parametrize("dtype", [BF, HALF, F32])
@pytest.mark.parametrize("m,h", [(400, 16384), (400, 9000), (310, 12345), (400, 8193), (303, 4097), (1000, 1026), (2500, 129)])
def test_many_wide_rows(cuda_device, dtype, m, h):
    check(*inputs(m, h, dtype, F32))


MANY = 500  # rows that go through the ring


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("h", [32, 96, 600, 2048, 3001, 9000])
def test_many_constant_rows(cuda_device, dtype, h):
    import mtp_b200
    x, w, b = inputs(MANY, h, dtype, F32)
    x[1::3], x[2::3] = 2.0, 0.0
    y = mtp_b200.layer_norm(x, w, b)
    want = b.to(dtype)
    # the sum of h twos is a number of fp32, and so is its quotient by h
    assert torch.equal(y[1::3], want.expand_as(y[1::3])) and torch.equal(y[2::3], want.expand_as(y[2::3]))
    check(x, w, b)
    with torch.no_grad():
        assert torch.isnan(mtp_b200.layer_norm(x, w, b, 0.0)[1::3]).all()  # 0 / 0, as the formula has it


@pytest.mark.parametrize("h", [64, 1024, 2048, 3000, 10000])
def test_offsets_of_many_rows_cost_no_digits(cuda_device, h):
    import mtp_b200
    x = (4096 + torch.arange(h, device="cuda") % 2).float()[None].repeat(MANY, 1)
    y = mtp_b200.layer_norm(x, eps=0.0)
    d = (h / 32 + 40) * U * 4096.5
    assert ((y.abs() - 1).abs() <= 4 * d + 16 * U).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("h", [48, 2048, 1001])
def test_bad_values_stay_in_their_row_of_many(cuda_device, bad, h):
    import mtp_b200
    x, w, b = inputs(MANY, h, F32, F32)
    clean = mtp_b200.layer_norm(x, w, b)
    x[77, 7] = bad
    x[401] = bad
    keep = torch.ones(MANY, dtype=torch.bool, device="cuda")
    keep[[77, 401]] = False
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = mtp_b200.layer_norm(*leaves)
    assert torch.isnan(y[~keep]).all() and torch.equal(y[keep], clean[keep])
    dx, dw, db = torch.autograd.grad(y, leaves, torch.ones_like(x))
    assert torch.isnan(dx[~keep]).all() and torch.isfinite(dx[keep]).all()
    assert torch.isnan(dw).all() and torch.isfinite(db).all()


def test_offsets_past_32_bits(cuda_device):
    """More than 2^31 values: the last rows are as in a call of their own."""
    import mtp_b200
    m, h = 1_050_000, 2048
    x = torch.zeros(m, h, dtype=BF, device="cuda")
    tail, w, b = inputs(600, h, BF, F32)
    x[-600:] = tail
    g = torch.zeros_like(x)
    g[-600:] = torch.randn(600, h, device="cuda").to(BF)
    results = []
    for rows, grad in ((x, g), (tail, g[-600:].clone())):
        leaves = [t.detach().requires_grad_() for t in (rows, w, b)]
        y = mtp_b200.layer_norm(*leaves)
        dx, dw, db = torch.autograd.grad(y, leaves, grad)
        results.append((y[-600:].detach().clone(), dx[-600:].clone(), dw, db))
        assert rows is tail or (torch.equal(y[0], b.to(BF)) and not dx[:-600].any())
        del y, dx
    for i in (0, 1):
        assert torch.equal(results[0][i], results[1][i])
    for i in (2, 3):  # 600 terms in another order
        size = g[-600:].abs().double().sum(0) * 8
        assert ((results[0][i].double() - results[1][i].double()).abs() <= 600 * U * size + 1e-6).all()

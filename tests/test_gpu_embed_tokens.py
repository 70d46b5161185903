"""Embedding rows and the table's gradient against the definition in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, HALF, F32, I32, I64 = torch.bfloat16, torch.float16, torch.float32, torch.int32, torch.int64
U = 2.0 ** -24


def half_step(t):
    i = torch.finfo(t)
    return i.eps / 2, i.smallest_normal * i.eps / 2


def check(ids, table, scale=1.0, grad=None):
    import mtp_b200
    v, h = table.shape
    table = table.detach().requires_grad_()
    out = mtp_b200.embed_tokens(ids, table, scale)
    assert out.shape == (*ids.shape, h) and out.dtype == table.dtype
    flat = ids.reshape(-1).long()
    inside = (flat >= 0) & (flat < v)
    want = torch.zeros(len(flat), h, dtype=torch.float64, device="cuda")
    want[inside] = scale * table.detach().double()[flat[inside]]
    rel, tiny = half_step(table.dtype)
    # one product in fp32 (of the scale's rounding too), one rounding
    assert ((out.detach().double().reshape(-1, h) - want).abs() <= (rel + 3 * U) * want.abs() + tiny).all()
    g = torch.randn(out.shape, device="cuda").to(table.dtype) if grad is None else grad
    (got,) = torch.autograd.grad(out, table, g)
    g64 = g.double().reshape(-1, h)[inside]
    total = torch.zeros(v, h, dtype=torch.float64, device="cuda").index_add_(0, flat[inside], g64)
    size = torch.zeros(v, h, dtype=torch.float64, device="cuda").index_add_(0, flat[inside], g64.abs())
    tokens = torch.bincount(flat[inside], minlength=v).double()[:, None]
    # a row's sum has at most as many additions as tokens; then the scale's rounding and one product
    bound = abs(scale) * ((tokens + 3) * U * size + rel * total.abs()) * (1 + 2 * rel) + tiny
    assert got.dtype == table.dtype and got.shape == table.shape
    error = (got.double() - scale * total).abs()
    assert (error <= bound).all(), float((error / (bound + 1e-300)).max())
    assert not got[tokens[:, 0] == 0].any()


def table_of(v, h, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(v, h, generator=g, device="cuda") / 8).to(dtype), g


SIZES = [(1, 1, 1), (1, 5, 64), (3, 2, 8), (16, 1, 40), (17, 3, 33), (64, 1000, 16), (511, 148, 100), (512, 149, 7), (513, 150, 24),
         (1000, 40, 2048), (2500, 7, 512), (4096, 5000, 128), (5000, 300, 1001), (3000, 2000, 4), (700, 131072, 8), (20000, 2, 64),
         (20000, 600, 6), (130, 90, 8192), (40000, 40000, 2)]


@pytest.mark.parametrize("n,v,h", SIZES)
@pytest.mark.parametrize("dtype", [BF, HALF, F32])
def test_sizes(cuda_device, n, v, h, dtype):
    table, g = table_of(v, h, dtype)
    check(torch.randint(0, v, (n,), generator=g, device="cuda", dtype=I32), table, 1.25)


@pytest.mark.parametrize("kind", [I32, I64])
@pytest.mark.parametrize("n", [40, 3000])
def test_ids_outside_the_table(cuda_device, kind, n):
    table, g = table_of(200, 48, F32)
    ids = torch.randint(-60, 260, (n,), generator=g, device="cuda", dtype=kind)
    ids[3] = torch.iinfo(kind).min
    ids[5] = torch.iinfo(kind).max
    ids[7] = -1
    check(ids, table)
    if kind == I64:
        ids[9] = 2 ** 32 + 4  # not row 4
        check(ids, table)
    check(torch.full((n,), -1, dtype=kind, device="cuda"), table)
    check(torch.full((n,), 200, dtype=kind, device="cuda"), table)


@pytest.mark.parametrize("n,v", [(5000, 3), (5000, 100000), (600, 1), (33000, 700), (20000, 262144)])
@pytest.mark.parametrize("h", [8, 520])
def test_one_row_for_most_tokens(cuda_device, n, v, h):
    """One id again and again (its sum reaches over many chunks), the others rare, and all ids close together."""
    table, g = table_of(v, h, BF)
    ids = torch.full((n,), v // 2, device="cuda", dtype=I32)
    ids[:: 37] = torch.randint(0, v, (len(ids[:: 37]),), generator=g, device="cuda", dtype=I32)
    check(ids, table)
    check(torch.randint(0, min(v, 900), (n,), generator=g, device="cuda", dtype=I32), table)
    check(torch.arange(n, device="cuda", dtype=I32) % v, table)
    check((torch.arange(n, device="cuda", dtype=I32) % v).flip(0).contiguous(), table)


def test_every_chunk_border(cuda_device):
    """Rows of one token to more than two chunks, begun at every place of a chunk."""
    table, _ = table_of(60, 16, F32)
    ids = torch.cat([torch.full((i,), i % 60) for i in range(60)]).to(device="cuda", dtype=I32)
    for shift in range(0, 17):
        check(torch.cat([torch.zeros(shift, dtype=I32, device="cuda"), ids]), table)


def test_sums_are_in_order(cuda_device):
    """Values whose sum depends on the order: as one after the other, ascending, for rows inside a chunk."""
    import mtp_b200
    table = torch.zeros(2, 8, device="cuda", requires_grad=True)
    ids = torch.tensor([1, 0, 1, 1], device="cuda", dtype=I32)
    g = torch.tensor([2.0 ** 25, 5.0, 1.0, -2.0 ** 25], device="cuda")[:, None].repeat(1, 8)
    (got,) = torch.autograd.grad(mtp_b200.embed_tokens(ids, table), table, g)
    assert got[1].tolist() == [0.0] * 8 and got[0].tolist() == [5.0] * 8


def test_shapes_of_ids(cuda_device):
    table, g = table_of(50, 24, F32)
    check(torch.randint(0, 50, (3, 4, 5), generator=g, device="cuda"), table)
    check(torch.tensor(7, device="cuda"), table)
    check(torch.zeros(0, dtype=I32, device="cuda"), table)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("h", [64, 130, 33])
def test_starts_off_16_bytes(cuda_device, dtype, h):
    table, g = table_of(90, h, dtype)
    buf = torch.empty(90 * h + 1, dtype=dtype, device="cuda")
    buf[1:] = table.flatten()
    ids = torch.randint(0, 90, (701,), generator=g, device="cuda", dtype=I32)
    grad = torch.empty(701 * h + 1, dtype=dtype, device="cuda").normal_()[1:].view(701, h)
    check(ids, buf[1:].view(90, h), 1.0, grad)


@pytest.mark.parametrize("scale", [0.0, -3.5, 45.254834, 1])
def test_scales(cuda_device, scale):
    table, g = table_of(64, 40, BF)
    check(torch.randint(0, 64, (300,), generator=g, device="cuda"), table, scale)


def test_infinities_stay_in_their_row(cuda_device):
    import mtp_b200
    table, g = table_of(30, 16, F32)
    ids = torch.randint(0, 29, (400,), generator=g, device="cuda", dtype=I32)
    ids[11] = 29
    grad = torch.randn(400, 16, generator=g, device="cuda")
    grad[11] = float("inf")
    table.requires_grad_()
    (got,) = torch.autograd.grad(mtp_b200.embed_tokens(ids, table), table, grad)
    assert torch.isinf(got[29]).all() and torch.isfinite(got[:29]).all()


def test_gradient_against_differences(cuda_device):
    import mtp_b200
    table, g = table_of(20, 8, F32)
    ids = torch.randint(-2, 20, (90,), generator=g, device="cuda")
    w = torch.randn(90, 8, generator=g, device="cuda")
    table.requires_grad_()
    (grad,) = torch.autograd.grad(mtp_b200.embed_tokens(ids, table, 1.5), table, w)
    d = torch.randn(20, 8, generator=g, device="cuda")
    with torch.no_grad():
        # linear: the difference of two calls, each rounded to 2 u of values below 8, h = 1
        up, down = (mtp_b200.embed_tokens(ids, table + s * d, 1.5).double() for s in (1, -1))
    slope = ((up - down) * w.double()).sum() / 2
    assert abs(float((grad.double() * d.double()).sum() - slope)) <= 90 * 8 * 16 * U * 8


@pytest.mark.parametrize("n,v", [(50000, 3000), (50000, 5)])
def test_same_bits_again(cuda_device, n, v):
    import mtp_b200
    table, g = table_of(v, 256, F32)
    table.requires_grad_()
    ids = torch.randint(0, v, (n,), generator=g, device="cuda", dtype=I32)
    grad = torch.randn(n, 256, generator=g, device="cuda")
    run = lambda: torch.autograd.grad(mtp_b200.embed_tokens(ids, table), table, grad)[0]
    first = run()
    for _ in range(3):
        assert torch.equal(run(), first)


def test_more_rows_than_a_slice_holds(cuda_device):
    """A table so long that a CTA takes its rows in two turns."""
    table, g = table_of(19_500_003, 1, F32)
    ids = torch.randint(0, 19_500_003, (3000,), generator=g, device="cuda", dtype=I32)
    ids[:600] = torch.arange(131_000, 131_600, device="cuda")  # over the turns' border
    ids[600:1300] = 131_100
    ids[1300] = 19_500_002
    check(ids, table, 0.5)


@pytest.mark.parametrize("n,v,h", [(1_300_000, 1000, 8), (600_000, 70, 40), (1_300_000, 300_000, 2)])
def test_very_many_tokens(cuda_device, n, v, h):
    table, g = table_of(v, h, F32)
    check(torch.randint(0, v, (n,), generator=g, device="cuda", dtype=I32), table)


@pytest.mark.parametrize("offset", [1, 2, 3])
@pytest.mark.parametrize("kind", [I32, I64])
def test_ids_off_16_bytes(cuda_device, kind, offset):
    table, g = table_of(500, 32, F32)
    ids = torch.randint(-3, 503, (2000 + offset,), generator=g, device="cuda", dtype=kind)[offset:]
    check(ids, table)


def test_offsets_past_32_bits(cuda_device):
    """More than 2^31 values in the table, in the rows and in the gradient."""
    import mtp_b200
    v = n = 1_050_000
    h = 2048
    table = torch.zeros(v, h, dtype=BF, device="cuda")
    table[-500:] = torch.randn(500, h, device="cuda").to(BF)
    ids = torch.zeros(n, dtype=I32, device="cuda")
    ids[-400:] = torch.arange(v - 400, v, device="cuda", dtype=I32)
    table.requires_grad_()
    out = mtp_b200.embed_tokens(ids, table)
    assert torch.equal(out[-400:].detach(), table[-400:].detach()) and not out[:-400].any()
    grad = torch.zeros_like(out)
    grad[-400:] = torch.randn(400, h, device="cuda").to(BF)
    grad[5] = 1
    (got,) = torch.autograd.grad(out, table, grad)
    assert torch.equal(got[-400:], grad[-400:]) and (got[0] == 1).all() and not got[1:-400].any()

"""sort_tokens / unsort_tokens against plain implementations: the sort bit for
bit, sums against 64 bits, gradients against their formulas and against
differences (both maps are linear in each input, so a difference is exact up to
rounding).

Tolerances: an fp32 sum of n products is within n * 2^-24 * sum|terms| of the
exact one whatever its order (one rounding per product and per addition, n + 1
of them used here), and a result of type T is then rounded once, by at most
2^-p(T) of itself (p = 8, 11, 24 bits for bf16, fp16, fp32)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def make_ids(g, m, k, e, none=0.0, low=None):
    ids = torch.rand(m, max(e, k), generator=g).argsort(-1)[:, :k].to(torch.int32) % e
    if none:
        ids[torch.rand(m, k, generator=g) < none] = -1
    if low is not None:
        ids[ids >= low] = low - 1  # a skewed routing: many pairs of one expert
    return ids


def plain_sort(ids, e, emap=None):
    """positions, pair of each row, offsets; plain Python counting."""
    flat = ids.flatten().tolist()
    if emap is not None:
        em = emap.tolist()
        flat = [em[i] if 0 <= i < len(em) else -1 for i in flat]
    keys = torch.tensor([i if 0 <= i < e else e for i in flat], dtype=torch.int64)
    pair = torch.sort(keys, stable=True).indices
    row = torch.empty_like(pair)
    row[pair] = torch.arange(len(pair))
    positions = torch.where(keys < e, row, ~row).to(torch.int32).view(ids.shape)
    offsets = torch.tensor([int((keys < v).sum()) for v in range(e + 1)], dtype=torch.int32)
    return positions, pair, offsets


def check_sort(x, ids, e, emap=None, scales=None, dev=None):
    import mtp_b200
    k = ids.shape[1]
    r = mtp_b200.sort_tokens(x, ids.to(dev), e, expert_map=None if emap is None else emap.to(dev),
                             row_scales=scales)
    positions, pair, offsets = plain_sort(ids, e, emap)
    assert torch.equal(r.positions.cpu(), positions)
    assert torch.equal(r.offsets.cpu(), offsets)
    rows = x.cpu()[pair // k].clone()
    rows[int(offsets[-1]):] = 0
    assert r.rows.shape == rows.shape and r.rows.dtype == x.dtype
    assert torch.equal(r.rows.cpu(), rows)
    if scales is None:
        assert r.row_scales is None
    else:
        s = scales.cpu()[pair // k].clone()
        s[int(offsets[-1]):] = 0
        assert torch.equal(r.row_scales.cpu(), s)
    return r


@pytest.mark.parametrize("m,k,e", [(0, 2, 4), (1, 1, 1), (1, 8, 256), (7, 3, 5), (64, 8, 256), (100, 32, 1024),
                                   (512, 8, 256), (513, 8, 256), (4097, 1, 3), (2048, 8, 1024), (3000, 7, 60),
                                   (8192, 8, 256), (20000, 8, 64), (70000, 4, 17)])
@pytest.mark.parametrize("none", [0.0, 0.6, 1.0])
def test_sort_bit_exact(cuda_device, m, k, e, none):
    g = torch.Generator().manual_seed(m * 31 + k + e)
    ids = make_ids(g, m, k, e, none)
    x = torch.randn(m, 24, generator=g).to(torch.bfloat16).to(cuda_device)
    check_sort(x, ids, e, dev=cuda_device)


def test_sort_skewed_and_out_of_range(cuda_device):
    g = torch.Generator().manual_seed(3)
    ids = make_ids(g, 5000, 6, 64, 0.1, low=2)
    ids[::7, 0] = 64            # one past the last expert
    ids[1::7, 1] = 2 ** 31 - 1
    ids[2::7, 2] = -(2 ** 31)
    x = torch.randn(5000, 16, generator=g).to(cuda_device)
    check_sort(x, ids, 64, dev=cuda_device)
    check_sort(x[:300], ids[:300], 64, dev=cuda_device)


@pytest.mark.parametrize("m", [40, 3000])
def test_sort_expert_map(cuda_device, m):
    g = torch.Generator().manual_seed(m)
    ids = make_ids(g, m, 4, 32, 0.05)
    emap = torch.full((32,), -1, dtype=torch.int32)
    emap[8:16] = torch.arange(8, dtype=torch.int32).flip(0)
    emap[3] = 900  # a local id past this rank's experts counts as none
    x = torch.randn(m, 40, generator=g).to(torch.float16).to(cuda_device)
    check_sort(x, ids, 8, emap, dev=cuda_device)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, torch.int8])
@pytest.mark.parametrize("h", [0, 1, 2, 3, 31, 64, 1000, 2048, 4100])
@pytest.mark.parametrize("m", [5, 1200])
def test_sort_widths_types_and_scales(cuda_device, dtype, h, m):
    g = torch.Generator().manual_seed(h + m)
    ids = make_ids(g, m, 4, 16, 0.2)
    x = (torch.randn(m, h, generator=g) * 40).to(dtype).to(cuda_device)
    check_sort(x, ids, 16, scales=torch.rand(m, generator=g).to(cuda_device), dev=cuda_device)


@pytest.mark.parametrize("m", [6, 1500])
def test_sort_strided_and_misaligned_rows(cuda_device, m):
    g = torch.Generator().manual_seed(m)
    ids = make_ids(g, m, 4, 16)
    wide = torch.randn(m, 100, generator=g).to(torch.bfloat16).to(cuda_device)
    check_sort(wide[:, 1:65], ids, 16, dev=cuda_device)   # 2-byte aligned start
    check_sort(wide[:, 8:72], ids, 16, dev=cuda_device)   # rows 200 bytes apart
    flat = torch.randn(m * 64 + 1, generator=g).to(torch.bfloat16).to(cuda_device)
    check_sort(flat[1:].view(m, 64), ids, 16, dev=cuda_device)


def weighted(m, k, h, e, dtype, none, seed, dev):
    import mtp_b200
    g = torch.Generator().manual_seed(seed)
    ids = make_ids(g, m, k, e, none)
    positions = plain_sort(ids, e)[0].to(dev)
    rows = torch.randn(m * k, h, generator=g).to(dtype).to(dev)
    w = torch.rand(m, k, generator=g).to(dev)
    grad = torch.randn(m, h, generator=g).to(dtype).to(dev)
    return mtp_b200, positions, rows, w, grad


def slots(positions):
    p = positions.long()
    return torch.where(p >= 0, p, ~p), (p >= 0)


CASES = [(1, 8, 2048, 256, 0.0), (1, 1, 1, 1, 0.0), (5, 3, 31, 7, 0.5), (64, 8, 2048, 256, 0.0),
         (33, 9, 100, 12, 0.3), (17, 32, 130, 64, 0.2), (700, 6, 1000, 60, 0.6), (2000, 8, 512, 256, 0.0),
         (9, 2, 5003, 4, 0.2), (50, 4, 64, 8, 1.0),
         # sizes that stream: one and two pieces a segment, short last segments, most slots and one more
         (3000, 8, 2048, 256, 0.1), (2500, 11, 1000, 60, 0.3), (5000, 2, 520, 16, 0.0), (2600, 1, 256, 4, 0.5),
         (2400, 12, 512, 32, 0.2), (2400, 22, 264, 64, 0.4), (2400, 23, 512, 64, 0.4), (2500, 5, 4104, 8, 0.2)]


def test_only_one_gradient(cuda_device):
    """Rows alone or weights alone, small and streamed: the same bits as both together."""
    for m in (40, 3000):
        pkg, positions, rows, w, grad = weighted(m, 8, 1024, 32, torch.bfloat16, 0.2, m, cuda_device)
        both = torch.autograd.grad(pkg.unsort_tokens(rows.requires_grad_(), positions, w.requires_grad_()), (rows, w), grad)
        rows, w = rows.detach(), w.detach()
        r, v = rows.clone().requires_grad_(), w.clone().requires_grad_()
        assert torch.equal(torch.autograd.grad(pkg.unsort_tokens(r, positions, w), r, grad)[0], both[0])
        assert torch.equal(torch.autograd.grad(pkg.unsort_tokens(rows, positions, v), v, grad)[0], both[1])


@pytest.mark.parametrize("m,k,h,e,none", CASES)
@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("with_weights", [True, False])
def test_unsort_and_gradients_against_64_bits(cuda_device, m, k, h, e, none, dtype, with_weights):
    pkg, positions, rows, w, grad = weighted(m, k, h, e, dtype, none, m + h, cuda_device)
    at, here = slots(positions)
    rows.requires_grad_()
    w = w.requires_grad_() if with_weights else None
    out = pkg.unsort_tokens(rows, positions, w)
    w64 = (w.detach().double() if with_weights else torch.ones(m, k, dtype=torch.float64, device=cuda_device)) * here
    picked = rows.detach().double()[at] * here[..., None]
    terms = picked * w64[..., None]
    ref = terms.sum(1)
    tol = (k + 1) * 2.0 ** -24 * terms.abs().sum(1) + U[dtype] * ref.abs() * (1 + 2.0 ** -6) + 1e-37
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25  # subnormal results
    assert ((out.detach().double() - ref).abs() <= tol).all()

    got = torch.autograd.grad(out, (rows, w) if with_weights else (rows,), grad)
    g64 = grad.double()
    ref_rows = torch.zeros(m * k, h, dtype=torch.float64, device=cuda_device)
    ref_rows[at.flatten()] = (g64[:, None] * w64[..., None]).flatten(0, 1)
    tol = (U[dtype] + 2.0 ** -23) * ref_rows.abs() + (2.0 ** -25 if dtype == torch.float16 else 1e-37)
    assert got[0].dtype == dtype
    assert ((got[0].double() - ref_rows).abs() <= tol).all()
    if with_weights:
        terms = picked * g64[:, None]
        tol = (h + 1) * 2.0 ** -24 * terms.abs().sum(-1) + 1e-37
        assert ((got[1].double() - terms.sum(-1)).abs() <= tol).all()


@pytest.mark.parametrize("m,k,h,e,none", CASES)
@pytest.mark.parametrize("dtype", list(U))
def test_sort_gradient_against_64_bits(cuda_device, m, k, h, e, none, dtype):
    import mtp_b200
    g = torch.Generator().manual_seed(m + k)
    ids = make_ids(g, m, k, e, none)
    x = torch.randn(m, h, generator=g).to(dtype).to(cuda_device).requires_grad_()
    r = mtp_b200.sort_tokens(x, ids.to(cuda_device), e)
    grad = torch.randn(m * k, h, generator=g).to(dtype).to(cuda_device)
    (gx,) = torch.autograd.grad(r.rows, x, grad)
    at, here = slots(r.positions)
    terms = grad.double()[at] * here[..., None]
    ref = terms.sum(1)
    tol = (k + 1) * 2.0 ** -24 * terms.abs().sum(1) + U[dtype] * ref.abs() * (1 + 2.0 ** -6) + 1e-37
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25
    assert gx.dtype == dtype
    assert ((gx.double() - ref).abs() <= tol).all()


def test_gradients_against_differences(cuda_device):
    """fp32; each map is linear in x, rows and w, so <f(v + d) - f(v), g> = <d, grad f>."""
    import mtp_b200
    g = torch.Generator().manual_seed(11)
    m, k, h, e = 37, 4, 96, 9
    ids = make_ids(g, m, k, e, 0.3).to(cuda_device)
    x, dx = (torch.randn(m, h, generator=g).to(cuda_device) for _ in range(2))
    w, dw = (torch.rand(m, k, generator=g).to(cuda_device) for _ in range(2))
    go = torch.randn(m, h, generator=g).to(cuda_device)

    def f(x, w):
        r = mtp_b200.sort_tokens(x, ids, e)
        return mtp_b200.unsort_tokens(r.rows, r.positions, w)

    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    gx, gw = torch.autograd.grad(f(xg, wg), (xg, wg), go)
    for (a, b, d, grad) in (((x + dx, w), (x, w), dx, gx), ((x, w + dw), (x, w), dw, gw)):
        diff = ((f(*a).double() - f(*b).double()) * go.double()).sum()
        want = (d.double() * grad.double()).sum()
        # every out element carries at most (k + 2) roundings of values below 30
        assert abs(diff - want) <= m * h * (k + 2) * 2.0 ** -24 * 30 * 2


def test_rows_of_nobody_are_not_read(cuda_device):
    """NaN in a row or weight of an unrouted pair stays there; infinities elsewhere go where they belong."""
    import mtp_b200
    ids = torch.tensor([[0, -1], [-1, -1], [1, 0]], dtype=torch.int32, device=cuda_device)
    x = torch.arange(3 * 8, dtype=torch.float32, device=cuda_device).view(3, 8)
    x[1] = float("nan")  # a token that no expert here takes
    r = mtp_b200.sort_tokens(x, ids, 2)
    assert torch.equal(r.positions.cpu(), torch.tensor([[0, ~3], [~4, ~5], [2, 1]], dtype=torch.int32))
    assert torch.equal(r.rows[3:], torch.zeros_like(r.rows[3:]))
    rows = r.rows.clone()
    rows[3:] = float("nan")
    w = torch.ones(3, 2, device=cuda_device)
    w[0, 1] = w[1, 0] = float("nan")
    rows.requires_grad_(), w.requires_grad_()
    out = mtp_b200.unsort_tokens(rows, r.positions, w)
    assert torch.equal(out[0], x[0]) and torch.equal(out[1], torch.zeros_like(out[1])) and torch.equal(out[2], 2 * x[2])
    g = torch.full((3, 8), float("inf"), device=cuda_device)
    g[2] = 1
    grows, gw = torch.autograd.grad(out, (rows, w), g)
    assert torch.equal(grows[3:], torch.zeros_like(grows[3:]))
    assert torch.isinf(grows[0]).all() and torch.equal(grows[1:3], torch.ones_like(grows[1:3]))
    assert gw[0, 1] == 0 and (gw[1] == 0).all() and gw[2, 0] == x[2].sum()


def test_gradient_forms_of_autograd(cuda_device):
    """Expanded and strided gradients, a second use of the inputs, only one input needing a gradient."""
    import mtp_b200
    g = torch.Generator().manual_seed(5)
    ids = make_ids(g, 20, 3, 6).to(cuda_device)
    x = torch.randn(20, 32, generator=g).to(cuda_device).requires_grad_()
    r = mtp_b200.sort_tokens(x, ids, 6)
    r.rows.sum().backward()  # a gradient of stride 0
    assert torch.equal(x.grad, torch.full_like(x, 3.0))
    w = torch.rand(20, 3, generator=g).to(cuda_device).requires_grad_()
    out = mtp_b200.unsort_tokens(r.rows.detach(), r.positions, w)
    out.t().square().sum().backward()
    want = torch.einsum("th,tkh->tk", 2 * out.detach().double(), r.rows.detach().double()[r.positions.long()])
    assert torch.allclose(w.grad.double(), want, rtol=1e-5, atol=1e-4)
    with torch.no_grad():
        assert not mtp_b200.unsort_tokens(r.rows, r.positions, w).requires_grad
    assert not r.positions.requires_grad and not r.offsets.requires_grad


def test_repeat_calls_and_streams_give_the_same_bits(cuda_device):
    import mtp_b200
    g = torch.Generator().manual_seed(8)
    ids = make_ids(g, 3000, 8, 128, 0.2).to(cuda_device)
    x = torch.randn(3000, 256, generator=g).to(torch.bfloat16).to(cuda_device)
    w = torch.rand(3000, 8, generator=g).to(cuda_device)

    def step():
        r = mtp_b200.sort_tokens(x, ids, 128)
        return r.rows, r.positions, r.offsets, mtp_b200.unsort_tokens(r.rows, r.positions, w)

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_rows_past_32_bit_offsets(cuda_device):
    """2.2e9 bytes of rows: byte offsets pass 2^31 (and element offsets 2^30)."""
    import mtp_b200
    m, k, h = 70000, 8, 2048
    g = torch.Generator(device=cuda_device).manual_seed(2)
    x = torch.randn(m, h, generator=g, device=cuda_device).to(torch.bfloat16)
    ids = torch.randint(0, 64, (m, k), generator=g, device=cuda_device, dtype=torch.int32)
    r = mtp_b200.sort_tokens(x, ids, 64)
    pair = torch.sort(ids.flatten().long(), stable=True).indices
    tail = pair[-1000:]
    assert torch.equal(r.rows[-1000:], x[tail // k])
    out = mtp_b200.unsort_tokens(r.rows, r.positions)
    assert torch.equal(out[-5000:], x[-5000:] * k)  # eight equal summands: exact

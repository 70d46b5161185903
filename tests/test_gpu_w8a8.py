"""int8 products against plain implementations in 64 bits (int8 products summed in
float64 are exact), quantisation bit for bit against the fp32 operations it is
defined by, the layer against its definition.

Tolerances: z = acc * sa * sb (+ bias) takes one rounding to fp32 for the sum and
one per operation, at most 4 * 2^-24 of |acc sa sb| + |bias|; the result is then
rounded once to its type (2^-8, 2^-11, 2^-24 of itself). silu(g) * u: the fast
exponential is off by 2 + 1.173 |g| units of 2^-23, the fast quotient by 2, the
sum and the two products by one each, and an error d of g moves silu by at most
(1 + |g|) d: together below (16 + 4 |g|) * 2^-23 relative."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def rounding(ref, dtype):
    t = U[dtype] * ref.abs() * (1 + 2.0 ** -6) + 1e-37
    return t + 2.0 ** -25 if dtype == torch.float16 else t


def check_product(out, acc, sa, sb, bias, dtype):
    z = acc * sa.double()[:, None] * sb.double()
    ref = z if bias is None else z + bias.double()
    tol = 2.0 ** -22 * (z.abs() + (0 if bias is None else bias.double().abs())) + rounding(ref, dtype)
    assert out.dtype == dtype and out.shape == ref.shape
    bad = (out.double() - ref).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}"


def codes(g, *shape, dev):
    return torch.randint(-128, 128, shape, generator=g, device=dev, dtype=torch.int8)


def scales(g, *shape, dev):
    return torch.rand(*shape, generator=g, device=dev) * 0.01 + 1e-4


# ---------------------------------------------------------------------------
# quantisation
# ---------------------------------------------------------------------------
def plain_codes(x):
    """The fp32 operations of the definition, in numpy."""
    x = x.float().cpu().numpy()
    most = np.abs(x).max(-1).astype(np.float32)
    pre = np.where(most < np.float32(2.0 ** -64), np.float32(2.0 ** 64), np.float32(1)).astype(np.float32)
    with np.errstate(divide="ignore"):
        factor = np.where(most > 0, np.float32(127) / (most * pre), np.float32(0)).astype(np.float32)
    q = np.rint((x * pre[:, None]).astype(np.float32) * factor[:, None]).astype(np.int8)
    return torch.from_numpy(q), torch.from_numpy(most / np.float32(127))


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("m,k", [(1, 1), (1, 2048), (3, 7), (5, 1001), (1, 70000), (64, 512), (1300, 64),
                                 (1500, 2049), (1200, 2056), (2000, 8), (0, 64)])
def test_quantize_bit_exact(cuda_device, dtype, m, k):
    import mtp_b200
    g = torch.Generator().manual_seed(m + k)
    x = torch.randn(m, k, generator=g) * torch.exp2(torch.randint(-12, 4, (m, 1), generator=g).float())
    if m > 2:
        x[1] = 0
        x[2] = x[2].sign()
    x = x.to(dtype)
    q, s = mtp_b200.quantize_int8(x.to(cuda_device))
    assert q.dtype == torch.int8 and q.shape == (m, k) and s.shape == (m,)
    if m:
        pq, ps = plain_codes(x)
        assert torch.equal(q.cpu(), pq)
        assert torch.equal(s.cpu(), ps)
        # half a step off at most (and what fp32 adds to a code of up to 127)
        err = (q.cpu().double() * s.cpu().double()[:, None] - x.double()).abs()
        assert (err <= s.cpu().double()[:, None] * (0.5 + 127 * 2.0 ** -22)).all()


def test_quantize_tiny_and_huge_rows(cuda_device):
    import mtp_b200
    x = torch.tensor([[1e-30, -2e-30, 0, 0.7e-30], [3e38, -1e38, 1, 0], [1e-38, -1e-39, 0, 0], [1e-45, 0, 0, 0]])
    q, s = mtp_b200.quantize_int8(x.to(cuda_device))
    pq, ps = plain_codes(x)
    assert torch.equal(q.cpu(), pq) and torch.equal(s.cpu(), ps)


@pytest.mark.parametrize("k", [16, 100, 4096])
def test_rows_with_infinities_and_nans_give_nan(cuda_device, k):
    import mtp_b200
    g = torch.Generator(device=cuda_device).manual_seed(k)
    x = torch.randn(4, k, generator=g, device=cuda_device)
    x[1, k // 2], x[2, 3], x[3, 0], x[3, 5] = float("inf"), float("nan"), float("-inf"), float("nan")
    q, s = mtp_b200.quantize_int8(x)
    assert not q[1:].any() and torch.isinf(s[1]) and torch.isnan(s[2]) and torch.isnan(s[3])
    w = codes(g, 24, k, dev=cuda_device)
    out = mtp_b200.int8_linear(x, w, scales(g, 24, dev=cuda_device))
    assert torch.isfinite(out[0]).all() and torch.isnan(out[1:]).all()


def test_quantize_strided_rows(cuda_device):
    import mtp_b200
    x = torch.randn(40, 300, device=cuda_device).to(torch.bfloat16)
    for part in (x[:, 8:136], x[:, 1:100], x[::2, :64]):
        q, s = mtp_b200.quantize_int8(part)
        pq, ps = plain_codes(part)
        assert torch.equal(q.cpu(), pq) and torch.equal(s.cpu(), ps)


# ---------------------------------------------------------------------------
# one product
# ---------------------------------------------------------------------------
SHAPES = [(1, 1, 1), (1, 1024, 2048), (2, 17, 16), (7, 129, 48), (8, 128, 31), (9, 200, 1001), (16, 64, 4096),
          (17, 1000, 256), (31, 33, 127), (33, 512, 128), (64, 2048, 512), (65, 130, 129), (100, 257, 2080),
          (128, 128, 128), (129, 300, 640), (255, 129, 96), (256, 256, 1024), (257, 1030, 272), (333, 517, 1001),
          (1000, 777, 336), (2048, 1024, 2048), (4100, 520, 144)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("with_bias", [False, True])
def test_int8_matmul(cuda_device, m, n, k, dtype, with_bias):
    import mtp_b200
    g = torch.Generator(device=cuda_device).manual_seed(m * 7 + n + k)
    a, b = codes(g, m, k, dev=cuda_device), codes(g, n, k, dev=cuda_device)
    sa, sb = scales(g, m, dev=cuda_device), scales(g, n, dev=cuda_device)
    bias = torch.randn(n, generator=g, device=cuda_device) if with_bias else None
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    out = mtp_b200.int8_matmul(a, sa, b, sb, bias=bias, out_dtype=dtype, status=status)
    check_product(out, a.double() @ b.double().T, sa, sb, bias, dtype)
    assert int(status) == 0


@pytest.mark.parametrize("m", [1, 5, 40, 300])
@pytest.mark.parametrize("sign", [-1, 1])
def test_extreme_codes_at_the_longest_k(cuda_device, m, sign):
    """-128 * -128 * K and -128 * 127 * K stay inside int32 for the longest K."""
    import mtp_b200
    k, n = 131071, 70
    a = torch.full((m, k), -128, dtype=torch.int8, device=cuda_device)
    b = torch.full((n, k), -128 if sign > 0 else 127, dtype=torch.int8, device=cuda_device)
    one_m, one_n = torch.ones(m, device=cuda_device), torch.ones(n, device=cuda_device)
    out = mtp_b200.int8_matmul(a, one_m, b, one_n, out_dtype=torch.float32)
    check_product(out, a.double() @ b.double().T, one_m, one_n, None, torch.float32)


@pytest.mark.parametrize("m,n,k", [(1, 1024, 2048), (5, 96, 100), (70, 517, 1001), (600, 256, 512)])
@pytest.mark.parametrize("dtype", list(U))
def test_int8_linear_is_quantize_then_matmul(cuda_device, m, n, k, dtype):
    import mtp_b200
    g = torch.Generator(device=cuda_device).manual_seed(m + n)
    x = torch.randn(m, k, generator=g, device=cuda_device).to(dtype)
    if m > 4:
        x[3] = 0
    w, sw = codes(g, n, k, dev=cuda_device), scales(g, n, dev=cuda_device)
    bias = torch.randn(n, generator=g, device=cuda_device)
    out = mtp_b200.int8_linear(x, w, sw, bias)
    q, s = mtp_b200.quantize_int8(x)
    check_product(out, q.double() @ w.double().T, s, sw, bias, dtype)
    assert torch.equal(out, mtp_b200.int8_matmul(q, s, w, sw, bias=bias, out_dtype=dtype))
    if m > 4:
        assert torch.equal(out[3], bias.to(dtype))
    assert mtp_b200.int8_linear(x, w, sw, out_dtype=torch.float32).dtype == torch.float32


def test_matmul_strided_and_misaligned_operands(cuda_device):
    import mtp_b200
    g = torch.Generator(device=cuda_device).manual_seed(1)
    for m in (3, 70):
        big = codes(g, m, 700, dev=cuda_device)
        flat = codes(g, 200 * 256 + 3, dev=cuda_device)
        sa = scales(g, m, dev=cuda_device)
        for a in (big[:, 16:272], big[:, 5:261], big[::2, :256]):
            for b in (flat[:-3].view(200, 256), flat[3:].view(200, 256), flat[1:-2].view(200, 256)):
                s, sb = sa[:a.shape[0]], scales(g, 200, dev=cuda_device)
                out = mtp_b200.int8_matmul(a, s, b, sb, out_dtype=torch.float32)
                check_product(out, a.double() @ b.double().T, s, sb, None, torch.float32)


# ---------------------------------------------------------------------------
# grouped products
# ---------------------------------------------------------------------------
GROUPS = [[1], [0, 3, 0], [5, 0, 1, 16, 17, 15], [256, 255, 257, 1, 0, 700], [0, 0, 0, 0], [1] * 40, [2000],
          [33, 64, 65, 128, 129, 31, 32], [8, 9, 7, 24, 25]]


def grouped_case(g, counts, tail, n, k, dev):
    p, e = sum(counts) + tail, len(counts)
    offsets = torch.tensor([0] + counts, dtype=torch.int32).cumsum(0).to(torch.int32).to(dev)
    a, b = codes(g, p, k, dev=dev), codes(g, e, n, k, dev=dev)
    return a, scales(g, p, dev=dev), b, scales(g, e, n, dev=dev), offsets


def grouped_acc(a, b, counts):
    acc = torch.zeros(a.shape[0], b.shape[1], dtype=torch.float64, device=a.device)
    at = 0
    for e, c in enumerate(counts):
        acc[at:at + c] = a[at:at + c].double() @ b[e].double().T
        at += c
    return acc


def row_group(counts, p, dev):
    r = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts))
    return torch.cat([r, torch.zeros(p - len(r), dtype=torch.int64)]).to(dev)


@pytest.mark.parametrize("counts", GROUPS)
@pytest.mark.parametrize("tail", [0, 13])
@pytest.mark.parametrize("n,k", [(128, 128), (100, 77), (1024, 512), (34, 272)])
@pytest.mark.parametrize("dtype", list(U))
def test_int8_grouped_matmul(cuda_device, counts, tail, n, k, dtype):
    import mtp_b200
    if sum(counts) + tail == 0:
        tail = 1
    g = torch.Generator(device=cuda_device).manual_seed(n + k + len(counts))
    a, sa, b, sb, offsets = grouped_case(g, counts, tail, n, k, cuda_device)
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    out = mtp_b200.int8_grouped_matmul(a, sa, b, sb, offsets, out_dtype=dtype, status=status)
    routed = sum(counts)
    acc, e = grouped_acc(a, b, counts), row_group(counts, a.shape[0], cuda_device)
    check_product(out[:routed], acc[:routed], sa[:routed], sb[e][:routed], None, dtype)
    assert not out[routed:].any()
    assert int(status) == 0


@pytest.mark.parametrize("counts", GROUPS)
@pytest.mark.parametrize("n,k", [(128, 128), (200, 77), (1024, 512), (34, 272), (2, 16)])
@pytest.mark.parametrize("dtype", list(U))
def test_int8_grouped_matmul_silu_mul(cuda_device, counts, n, k, dtype):
    import mtp_b200
    g = torch.Generator(device=cuda_device).manual_seed(n + k + len(counts))
    a, sa, b, sb, offsets = grouped_case(g, counts, 5, n, k, cuda_device)
    sa = sa / (k ** 0.5 / 4)
    out = mtp_b200.int8_grouped_matmul(a, sa, b, sb, offsets, out_dtype=dtype, activation="silu_mul")
    routed, e = sum(counts), row_group(counts, a.shape[0], cuda_device)
    z = grouped_acc(a, b, counts) * sa.double()[:, None] * sb.double()[e]
    gate, up = z[:, :n // 2], z[:, n // 2:]
    ref = (gate * torch.sigmoid(gate) * up)[:routed]
    tol = (16 + 4 * gate[:routed].abs()) * 2.0 ** -23 * ref.abs() + rounding(ref, dtype) + 1e-30
    assert out.shape == (a.shape[0], n // 2) and out.dtype == dtype
    assert ((out[:routed].double() - ref).abs() <= tol).all()
    assert not out[routed:].any()


@pytest.mark.parametrize("counts,n", [([3000, 2500, 2700], 512), ([900, 1, 1100], 520), ([300] * 40, 200)])
@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("activation", [None, "silu_mul"])
def test_grouped_large_groups(cuda_device, counts, n, dtype, activation):
    """Groups of several tiles of the larger sizes, gated and not."""
    import mtp_b200
    g = torch.Generator(device=cuda_device).manual_seed(n + len(counts))
    a, sa, b, sb, offsets = grouped_case(g, counts, 70, n, 400, cuda_device)
    sa = sa / 5
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    out = mtp_b200.int8_grouped_matmul(a, sa, b, sb, offsets, out_dtype=dtype, activation=activation, status=status)
    routed, e = sum(counts), row_group(counts, a.shape[0], cuda_device)
    acc = grouped_acc(a, b, counts)
    if activation is None:
        check_product(out[:routed], acc[:routed], sa[:routed], sb[e][:routed], None, dtype)
    else:
        z = (acc * sa.double()[:, None] * sb.double()[e])[:routed]
        gate, up = z[:, :n // 2], z[:, n // 2:]
        ref = gate * torch.sigmoid(gate) * up
        tol = (16 + 4 * gate.abs()) * 2.0 ** -23 * ref.abs() + rounding(ref, dtype) + 1e-30
        assert ((out[:routed].double() - ref).abs() <= tol).all()
    assert not out[routed:].any() and int(status) == 0


@pytest.mark.parametrize("rows", [12, 900])
def test_grouped_rows_of_no_group(cuda_device, rows):
    """Rows before offsets[0] are zeros, offsets past the rows are clamped."""
    import mtp_b200
    g = torch.Generator(device=cuda_device).manual_seed(rows)
    a, b = codes(g, rows, 64, dev=cuda_device), codes(g, 3, 40, 64, dev=cuda_device)
    sa, sb = scales(g, rows, dev=cuda_device), scales(g, 3, 40, dev=cuda_device)
    mid = rows // 2
    offsets = torch.tensor([5, mid, mid, rows + 7], dtype=torch.int32, device=cuda_device)
    out = mtp_b200.int8_grouped_matmul(a, sa, b, sb, offsets, out_dtype=torch.float32)
    assert not out[:5].any()
    for e, part in ((0, slice(5, mid)), (2, slice(mid, rows))):
        check_product(out[part], a[part].double() @ b[e].double().T, sa[part], sb[e], None, torch.float32)


def test_grouped_many_experts_and_64_bit_offsets(cuda_device):
    """1024 groups; weights of 2.1e9 bytes, so that their byte offsets pass 2^31."""
    import mtp_b200
    g = torch.Generator(device=cuda_device).manual_seed(4)
    counts = [0] * 1024
    counts[0], counts[511], counts[1000], counts[1023] = 3, 40, 1, 20
    a, sa, b, sb, offsets = grouped_case(g, counts, 0, 1024, 2048, cuda_device)
    out = mtp_b200.int8_grouped_matmul(a, sa, b, sb, offsets, out_dtype=torch.float32)
    e = row_group(counts, a.shape[0], cuda_device)
    check_product(out, grouped_acc(a, b, counts), sa, sb[e], None, torch.float32)


def test_output_past_32_bit_offsets(cuda_device):
    import mtp_b200
    m, n, k = 70000, 16400, 32
    g = torch.Generator(device=cuda_device).manual_seed(9)
    a, b = codes(g, m, k, dev=cuda_device), codes(g, n, k, dev=cuda_device)
    sa, sb = scales(g, m, dev=cuda_device), scales(g, n, dev=cuda_device)
    out = mtp_b200.int8_matmul(a, sa, b, sb, out_dtype=torch.float32)
    check_product(out[-300:], a[-300:].double() @ b.double().T, sa[-300:], sb, None, torch.float32)


def test_repeat_calls_streams_and_graphs_give_the_same_bits(cuda_device):
    import mtp_b200
    g = torch.Generator(device=cuda_device).manual_seed(6)
    x = torch.randn(300, 512, generator=g, device=cuda_device).to(torch.bfloat16)
    w, sw = codes(g, 700, 512, dev=cuda_device), scales(g, 700, dev=cuda_device)
    first = mtp_b200.int8_linear(x, w, sw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = mtp_b200.int8_linear(x, w, sw)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, second)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = mtp_b200.int8_linear(x, w, sw)
    x.mul_(-1)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(third, -first)


# ---------------------------------------------------------------------------
# the layer
# ---------------------------------------------------------------------------
def layer_case(g, m, e, h, i, dtype, dev):
    return dict(x=torch.randn(m, h, generator=g, device=dev).to(dtype),
                logits=torch.randn(m, e, generator=g, device=dev),
                w13=codes(g, e, 2 * i, h, dev=dev), s13=(0.5 + torch.rand(e, 2 * i, generator=g, device=dev)) / (73 * h ** 0.5),
                w2=codes(g, e, h, i, dev=dev), s2=(0.5 + torch.rand(e, h, generator=g, device=dev)) / (73 * i ** 0.5))


def codes64(x):
    most = x.abs().amax(-1, keepdim=True)
    return torch.where(most > 0, torch.round(127 * x / most), 0.0), most[:, 0] / 127


def plain_layer(c, w, ids):
    """The definition in 64 bits; ids outside [0, E) contribute nothing."""
    x = c["x"].double()
    out = torch.zeros_like(x)
    q, s = codes64(x)
    for e in range(c["w13"].shape[0]):
        t, j = (ids == e).nonzero(as_tuple=True)
        if not len(t):
            continue
        z = q[t] @ c["w13"][e].double().T * s[t, None] * c["s13"][e].double()
        gate, up = z.chunk(2, -1)
        hq, hs = codes64(gate * torch.sigmoid(gate) * up)
        y = hq @ c["w2"][e].double().T * hs[:, None] * c["s2"][e].double()
        out.index_add_(0, t, y * w.double()[t, j, None])
    return out


def check_layer(out, ref):
    """The bars of the package's layer outputs: rel-L2 1e-2, max-abs 2e-2 of the largest. (Each pair's
    output and the result are rounded to the 8 or 11 bits of their type, 2^-8 = 3.9e-3 at most each; a
    code that falls the other way at a tie moves its row by 1/127 of its largest element, on few rows.)"""
    d = out.double() - ref
    assert d.norm() <= 1e-2 * ref.norm()
    assert d.abs().max() <= 2e-2 * max(1.0, float(ref.abs().max()))


@pytest.mark.parametrize("m,e,k,h,i", [(1, 256, 8, 512, 128), (4, 8, 2, 256, 128), (33, 16, 4, 272, 96),
                                       (300, 32, 8, 512, 256), (1025, 8, 3, 128, 64), (50, 5, 2, 100, 30),
                                       (2, 1024, 8, 64, 48), (7, 1, 1, 48, 16),
                                       (8, 64, 32, 256, 64), (1, 4, 2, 2048, 1024), (3, 6, 2, 4096, 16), (6, 300, 4, 80, 528)])
@pytest.mark.parametrize("dtype", list(U))
def test_layer_against_its_definition(cuda_device, m, e, k, h, i, dtype):
    import mtp_b200
    g = torch.Generator(device=cuda_device).manual_seed(m + e)
    c = layer_case(g, m, e, h, i, dtype, cuda_device)
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    out = mtp_b200.moe_layer_w8a8(c["x"], c["logits"], c["w13"], c["s13"], c["w2"], c["s2"], k, status=status)
    w, ids, _ = mtp_b200.topk_softmax(c["logits"], k)
    check_layer(out, plain_layer(c, w, ids))
    assert int(status) == 0
    given = mtp_b200.moe_layer_w8a8(c["x"], None, c["w13"], c["s13"], c["w2"], c["s2"], k, topk_weights=w, topk_ids=ids)
    assert torch.equal(given, out)


@pytest.mark.parametrize("m", [1, 5, 8, 9, 40])
def test_layer_with_many_pairs_of_one_expert(cuda_device, m):
    """Given ids: an expert several times in one token (more than 8 pairs in all), ids of nobody, a token without any."""
    import mtp_b200
    g = torch.Generator(device=cuda_device).manual_seed(m)
    c = layer_case(g, m, 5, 160, 48, torch.bfloat16, cuda_device)
    ids = torch.randint(-1, 6, (m, 7), generator=g, device=cuda_device, dtype=torch.int32)
    ids[:, :3] = 2
    ids[m // 2] = -1
    w = torch.rand(m, 7, generator=g, device=cuda_device) / 7
    out = mtp_b200.moe_layer_w8a8(c["x"], None, c["w13"], c["s13"], c["w2"], c["s2"], 7, topk_weights=w, topk_ids=ids)
    check_layer(out, plain_layer(c, w, ids))
    assert not out[m // 2].any()


@pytest.mark.parametrize("m", [4, 60, 700])
def test_layer_keeps_a_bad_token_to_itself(cuda_device, m):
    """An infinity or a NaN in one token's row makes that token's output NaN and no other's."""
    import mtp_b200
    g = torch.Generator(device=cuda_device).manual_seed(m)
    c = layer_case(g, m, 8, 128, 64, torch.bfloat16, cuda_device)
    args = (c["logits"], c["w13"], c["s13"], c["w2"], c["s2"], 2)
    good = mtp_b200.moe_layer_w8a8(c["x"], *args)
    x = c["x"].clone()
    x[1, 7], x[m - 1, 0] = float("nan"), float("inf")
    out = mtp_b200.moe_layer_w8a8(x, *args)
    bad = torch.zeros(m, dtype=torch.bool, device=cuda_device)
    bad[1] = bad[m - 1] = True
    assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], good[~bad])


def test_layer_in_a_graph_and_on_a_side_stream(cuda_device):
    import mtp_b200
    for m in (2, 30):
        g = torch.Generator(device=cuda_device).manual_seed(m)
        c = layer_case(g, m, 16, 256, 128, torch.bfloat16, cuda_device)
        call = lambda: mtp_b200.moe_layer_w8a8(c["x"], c["logits"], c["w13"], c["s13"], c["w2"], c["s2"], 4)
        first = call()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            second = call()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                third = call()
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(first, second)
        c["x"].mul_(-1)
        want = call()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(third, want)


@pytest.mark.parametrize("m", [3, 400])
def test_layer_expert_shards_add_up(cuda_device, m):
    """Two ranks' shards through expert_map; ids of nobody and rows without a pair contribute nothing."""
    import mtp_b200
    g = torch.Generator(device=cuda_device).manual_seed(m)
    c = layer_case(g, m, 8, 256, 64, torch.float32, cuda_device)
    w, ids, _ = mtp_b200.topk_softmax(c["logits"], 3)
    ids[0] = -1
    ids[1, 1] = 8
    whole = mtp_b200.moe_layer_w8a8(c["x"], None, c["w13"], c["s13"], c["w2"], c["s2"], 3, topk_weights=w, topk_ids=ids)
    check_layer(whole, plain_layer(c, w, ids))
    assert not whole[0].any()
    parts = torch.zeros_like(whole)
    for r in range(2):
        emap = torch.full((8,), -1, dtype=torch.int32, device=cuda_device)
        emap[4 * r:4 * r + 4] = torch.arange(4, dtype=torch.int32, device=cuda_device)
        mine = slice(4 * r, 4 * r + 4)
        parts += mtp_b200.moe_layer_w8a8(c["x"], None, c["w13"][mine], c["s13"][mine], c["w2"][mine], c["s2"][mine], 3,
                                         topk_weights=w, topk_ids=ids, expert_map=emap)
    # the same fp32 products, added in another order
    assert ((parts - whole).abs() <= 8 * 2.0 ** -24 * (whole.abs() + whole.abs().max())).all()


def test_layer_empty_batch_and_out(cuda_device):
    import mtp_b200
    g = torch.Generator(device=cuda_device).manual_seed(1)
    c = layer_case(g, 6, 4, 64, 32, torch.bfloat16, cuda_device)
    args = (c["w13"], c["s13"], c["w2"], c["s2"], 2)
    assert mtp_b200.moe_layer_w8a8(c["x"][:0], c["logits"][:0], *args).shape == (0, 64)
    out = torch.empty_like(c["x"])
    assert mtp_b200.moe_layer_w8a8(c["x"], c["logits"], *args, out=out) is out
    assert torch.equal(out, mtp_b200.moe_layer_w8a8(c["x"], c["logits"], *args))

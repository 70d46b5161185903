"""SiLU(gate) * up of fp32 results: a few units in the last place whatever the gate.

The gates are exact in fp32 (whole codes times powers of two, so neither the sum nor the scales round). expf is
within 1 unit in the last place of fp32 (2^-23 of a value at most) and the fast quotient within 2, 1 + expf and the
product with up round by half a unit each: together 4 * 2^-23, and what they compound. The quotient is zero where the
exponential passes 2^126: gates from -87.4 down, silu below 2^-119."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def reference(gate, up):
    """(result, tolerance) in 64 bits."""
    r = gate / (1 + torch.exp(-gate)) * up
    return r, 4 * 2.0 ** -23 * (1 + 2.0 ** -10) * r.abs() + 2.0 ** -119 * up.abs()


@pytest.mark.parametrize("rows", [7, 60, 900])
@pytest.mark.parametrize("step", [1.0, 0.125, 0.0078125])
def test_gated_fp32_products(cuda_device, rows, step):
    import mtp_b200
    g = torch.Generator(device=cuda_device).manual_seed(rows)
    n, k = 64, 32
    a = torch.zeros(rows, k, dtype=torch.int8, device=cuda_device)
    a[:, 0] = torch.randint(-120, 121, (rows,), generator=g, device=cuda_device)
    a[:, 1] = torch.randint(1, 5, (rows,), generator=g, device=cuda_device)
    b = torch.zeros(2, 2 * n, k, dtype=torch.int8, device=cuda_device)
    b[:, :n, 0] = 1
    b[:, n:, 1] = torch.randint(-7, 8, (2, n), generator=g, device=cuda_device)
    offsets = torch.tensor([0, rows // 3, rows], dtype=torch.int32, device=cuda_device)
    sb = torch.ones(2, 2 * n, device=cuda_device)
    sb[:, :n] = step
    out = mtp_b200.int8_grouped_matmul(a, torch.ones(rows, device=cuda_device), b, sb, offsets, out_dtype=torch.float32,
                                       activation="silu_mul")
    group = (torch.arange(rows, device=cuda_device) >= rows // 3).long()
    up = a[:, 1, None].double() * b[group, n:, 1].double()
    ref, tol = reference((a[:, 0, None].double() * step).expand(rows, n), up)
    assert ((out.double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("m", [2, 40])
def test_layer_h_by_its_scale(cuda_device, m):
    """One channel of h, one of the result: code 127 exactly, so the result is h within the roundings of
    max / 127, two scales of one, the weighted sum (2 products) on top."""
    import mtp_b200
    g = torch.Generator(device=cuda_device).manual_seed(m)
    h = i = 16
    x = torch.zeros(m, h, device=cuda_device)
    x[:, 0] = 127                                                 # scale 1, codes as they are
    x[:, 1] = torch.randint(-85, 86, (m,), generator=g, device=cuda_device).float()
    x[0, 1], x[1, 1] = -84, -60
    w13 = torch.zeros(1, 2 * i, h, dtype=torch.int8, device=cuda_device)
    w13[0, 0, 1], w13[0, i, 0] = 1, 1
    w2 = torch.zeros(1, h, i, dtype=torch.int8, device=cuda_device)
    w2[0, :, 0] = 1
    one = torch.ones(m, 1, device=cuda_device)
    ids = torch.zeros(m, 1, dtype=torch.int32, device=cuda_device)
    out = mtp_b200.moe_layer_w8a8(x, None, w13, torch.ones(1, 2 * i, device=cuda_device), w2,
                                  torch.ones(1, h, device=cuda_device), 1, topk_weights=one, topk_ids=ids)
    ref, tol = reference(x[:, 1].double(), torch.full((m,), 127.0, dtype=torch.float64, device=cuda_device))
    assert ((out.double() - ref[:, None]).abs() <= tol[:, None] + 4 * 2.0 ** -24 * ref.abs()[:, None]).all()

"""The W8A8 layer holds h and each pair's down output in fp32, whatever its type and the number of its tokens.

Against the definition in 64 bits, element by element. The kernel's h is off by at most
e = (16 + 4 |gate|) * 2^-23 of itself (fast or precise exponential; see test_gpu_w8a8.py), so its codes may
differ from those of the 64-bit h only where 127 h / max|h| lies within 127 e(h) + 127 e(max) + 127 * 3 * 2^-24
(the division, the product and the maximum's rounding) of a tie, there by one: |w2| * scale each. The scale is off
by e(max) + 2^-24, the product takes 4 roundings to fp32, the weighted sum one per pair and one more, and the
result is rounded once to its type."""
import pytest
import torch

from test_gpu_w8a8 import layer_case, rounding

E24 = 2.0 ** -24


def reference(q, s, c, w, ids, h_type=torch.float64, y_type=torch.float64):
    """(result in 64 bits, bound of a kernel's fp32 error) of the layer for rows q with scales s. h_type and y_type:
    narrower types to hold h and the pairs' down outputs in."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for e in range(c["w13"].shape[0]):
        t, j = (ids == e).nonzero(as_tuple=True)
        if not len(t):
            continue
        z = q[t].double() @ c["w13"][e].double().T * s.double()[t, None] * c["s13"][e].double()
        gate, up = z.chunk(2, -1)
        h = (gate * torch.sigmoid(gate) * up).to(h_type).double()
        off = (16 + 4 * gate.abs()) * 2 * E24
        most, at = h.abs().max(-1, keepdim=True)
        off_most = off.gather(1, at)
        place = 127 * h / most.clamp(min=1e-300)
        near = (place - torch.floor(place) - 0.5).abs() <= place.abs() * (off + off_most + 3 * E24)
        w2, scale = c["w2"][e].double(), most / 127 * c["s2"][e].double()
        y = (torch.round(place) @ w2.T * scale).to(y_type).double()
        pair = w.double()[t, j, None]
        out.index_add_(0, t, y * pair)
        miss = near.double() @ w2.abs().T * scale + y.abs() * (off_most + 6 * E24)
        bound.index_add_(0, t, (miss + y.abs() * (ids.shape[1] + 1) * E24) * pair.abs())
    return out, bound


@pytest.mark.gpu
@pytest.mark.parametrize("m,e,k,h,i", [(1, 16, 4, 512, 128), (4, 8, 2, 256, 128), (8, 64, 32, 256, 64), (9, 8, 2, 256, 128),
                                       (33, 16, 4, 272, 96), (50, 5, 2, 100, 30), (300, 32, 8, 512, 256), (700, 4, 3, 1000, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_layer_error_is_that_of_fp32(cuda_device, m, e, k, h, i, dtype):
    import mtp_b200
    g = torch.Generator(device=cuda_device).manual_seed(m + h)
    c = layer_case(g, m, e, h, i, dtype, cuda_device)
    w, ids, _ = mtp_b200.topk_softmax(c["logits"], k)
    out = mtp_b200.moe_layer_w8a8(c["x"], c["logits"], c["w13"], c["s13"], c["w2"], c["s2"], k)
    ref, bound = reference(*mtp_b200.quantize_int8(c["x"]), c, w, ids)
    bad = (out.double() - ref).abs() > bound + rounding(ref.abs() + bound, dtype)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("h,i", [(128, 64), (1024, 256)])
def test_layer_gives_a_token_the_same_bits_in_every_batch(cuda_device, dtype, h, i):
    import mtp_b200
    g = torch.Generator(device=cuda_device).manual_seed(h)
    m = 1300  # the few-token kernels, the row loops of unsort and its bulk copies
    c = layer_case(g, m, 8, h, i, dtype, cuda_device)
    args = (c["w13"], c["s13"], c["w2"], c["s2"], 3)
    layer = lambda part: mtp_b200.moe_layer_w8a8(c["x"][part].contiguous(), c["logits"][part].contiguous(), *args)
    whole = layer(slice(0, m))
    for n in (1, 4, 8, 9, 100):
        assert torch.equal(layer(slice(0, n)), whole[:n]), n
    assert torch.equal(layer(slice(m - 5, m)), whole[m - 5:])


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 32, 1300])
def test_fp16_layer_with_pairs_past_the_range_of_fp16(cuda_device, m):
    """Down outputs beyond 65504 with small weights: the weighted sum is a number."""
    import mtp_b200
    g = torch.Generator(device=cuda_device).manual_seed(m)
    c = layer_case(g, m, 8, 512, 64, torch.float16, cuda_device)
    c["s2"] = c["s2"] * 3e5
    ids = torch.rand(m, 8, generator=g, device=cuda_device).argsort(-1)[:, :2].to(torch.int32).contiguous()
    w = torch.full((m, 2), 1e-4, device=cuda_device)
    w[:, 1] = 0
    out = mtp_b200.moe_layer_w8a8(c["x"], None, c["w13"], c["s13"], c["w2"], c["s2"], 2, topk_weights=w, topk_ids=ids)
    ref, bound = reference(*mtp_b200.quantize_int8(c["x"]), c, w, ids)
    assert float(ref.abs().max()) * 1e4 > 65504 and float(ref.abs().max()) < 65504
    assert ((out.double() - ref).abs() <= bound + rounding(ref.abs() + bound, torch.float16)).all()


@pytest.mark.parametrize("narrow", ["h_type", "y_type"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_the_bound_sees_16_bit_intermediates(narrow, dtype):
    """On the CPU: the definition with h or the down outputs rounded to 16 bits is outside the bound of an fp32 layer."""
    g = torch.Generator().manual_seed(3)
    c = layer_case(g, 20, 4, 96, 64, torch.float32, "cpu")
    s = c["x"].abs().amax(-1) / 127
    q = torch.round(c["x"] / s[:, None])
    ids = torch.randint(0, 4, (20, 2), generator=g, dtype=torch.int32)
    w = torch.rand(20, 2, generator=g)
    ref, bound = reference(q, s, c, w, ids)
    out, _ = reference(q, s, c, w, ids, **{narrow: dtype})
    assert ((out - ref).abs() > bound + rounding(ref.abs() + bound, torch.float32)).double().mean() > 0.05

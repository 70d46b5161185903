"""The int8 functions have no gradients: with inputs that require one they give their results, and a backward pass
through them, or a forward-mode derivative, is an error and not a missing term."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu

I8, I32 = torch.int8, torch.int32


def cases(dev):
    """name -> (call of a dict of the floating inputs, that dict)"""
    import mtp_b200 as p
    g = torch.Generator(device=dev).manual_seed(0)
    f = lambda *s: torch.rand(*s, generator=g, device=dev) + 0.1
    q = lambda *s: torch.randint(-127, 128, s, generator=g, device=dev, dtype=I8)
    a, b, b3 = q(6, 32), q(8, 32), q(2, 8, 32)
    offsets = torch.tensor([0, 2, 6], dtype=I32, device=dev)
    w13, w2 = q(3, 16, 32), q(3, 32, 8)
    ids = torch.randint(0, 3, (6, 2), generator=g, device=dev, dtype=I32)
    return {
        "quantize_int8": (lambda t: p.quantize_int8(t["x"])[1], dict(x=f(6, 30))),
        "int8_matmul": (lambda t: p.int8_matmul(a, t["sa"], b, t["sb"], bias=t["bias"], out_dtype=torch.float32),
                        dict(sa=f(6), sb=f(8), bias=f(8))),
        "int8_linear": (lambda t: p.int8_linear(t["x"], b, t["sb"], t["bias"]), dict(x=f(6, 32), sb=f(8), bias=f(8))),
        "int8_grouped_matmul": (lambda t: p.int8_grouped_matmul(a, t["sa"], b3, t["sb"], offsets, out_dtype=torch.float32),
                                dict(sa=f(6), sb=f(2, 8))),
        "moe_layer_w8a8": (lambda t: p.moe_layer_w8a8(t["x"], t["logits"], w13, t["s13"], w2, t["s2"], 2),
                           dict(x=f(6, 32), logits=f(6, 3), s13=f(3, 16), s2=f(3, 32))),
        "moe_layer_w8a8 of given ids": (
            lambda t: p.moe_layer_w8a8(t["x"], None, w13, t["s13"], w2, t["s2"], 2, topk_weights=t["w"], topk_ids=ids),
            dict(x=f(6, 32), w=f(6, 2), s13=f(3, 16), s2=f(3, 32))),
        "row_scales of sort_tokens": (lambda t: p.sort_tokens(a, ids, 3, row_scales=t["s"]).row_scales, dict(s=f(6))),
    }


NAMES = ["quantize_int8", "int8_matmul", "int8_linear", "int8_grouped_matmul", "moe_layer_w8a8", "moe_layer_w8a8 of given ids",
         "row_scales of sort_tokens"]


@pytest.mark.parametrize("name", NAMES)
def test_backward_raises_for_every_input(cuda_device, name):
    call, inputs = cases(cuda_device)[name]
    want = call(inputs)
    assert not want.requires_grad
    for key in inputs:
        t = {k: v.clone().requires_grad_(k == key) for k, v in inputs.items()}
        out = call(t)
        assert torch.equal(out, want) and out.requires_grad, key
        with pytest.raises(NotImplementedError, match=name.split(" of given")[0]):
            (out * 2).sum().backward()
        with torch.no_grad():
            assert not call(t).requires_grad
        out.detach_().mul_(2)  # the result is the caller's own


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_raises_for_every_input(cuda_device, name):
    call, inputs = cases(cuda_device)[name]
    for key in inputs:
        with forward_ad.dual_level():
            t = {k: forward_ad.make_dual(v, torch.ones_like(v)) if k == key else v for k, v in inputs.items()}
            with pytest.raises(NotImplementedError):
                call(t)


def test_layer_with_out_and_a_gradient(cuda_device):
    import mtp_b200
    x, lg = torch.zeros(2, 32, device=cuda_device), torch.zeros(2, 3, device=cuda_device)
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device=cuda_device)
    args = (z(3, 16, 32, dtype=I8), z(3, 16), z(3, 32, 8, dtype=I8), z(3, 32), 2)
    out = torch.empty_like(x)
    with pytest.raises(RuntimeError, match="out"):
        mtp_b200.moe_layer_w8a8(x.requires_grad_(), lg, *args, out=out)
    with torch.no_grad():
        assert mtp_b200.moe_layer_w8a8(x, lg, *args, out=out) is out
    assert not out.requires_grad

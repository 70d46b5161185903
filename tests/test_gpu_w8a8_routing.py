"""Tokens with NaN logits in the W8A8 layer: their output is NaN, the other tokens keep theirs, whatever the
width and alignment of the rows and the number of tokens."""
import pytest
import torch

from test_gpu_w8a8 import layer_case

pytestmark = pytest.mark.gpu

NAN = float("nan")


@pytest.mark.parametrize("m", [3, 8, 9, 60, 1300])
@pytest.mark.parametrize("h", [100, 101, 128, 264])
@pytest.mark.parametrize("e", [8, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_nan_logits_give_nan(cuda_device, m, h, e, dtype):
    import mtp_b200
    g = torch.Generator(device=cuda_device).manual_seed(m + h)
    c = layer_case(g, m, e, h, 48, dtype, cuda_device)
    layer = lambda logits: mtp_b200.moe_layer_w8a8(c["x"], logits, c["w13"], c["s13"], c["w2"], c["s2"], 4)
    good = layer(c["logits"])
    assert torch.isfinite(good).all()
    logits = c["logits"].clone()
    logits[0] = NAN            # a token whose hidden state was NaN
    logits[1, e // 2] = NAN    # one expert's alone
    logits[m - 1, 2:] = NAN    # fewer numbers than choices
    out = layer(logits)
    bad = torch.zeros(m, dtype=torch.bool, device=cuda_device)
    bad[[0, 1, m - 1]] = True
    assert torch.isnan(out[bad]).all()
    assert torch.equal(out[~bad], good[~bad])


@pytest.mark.parametrize("m", [3, 60])
@pytest.mark.parametrize("h", [100, 101, 128])
@pytest.mark.parametrize("e", [5, 40, 300])
def test_routes_as_topk_softmax_does(cuda_device, m, h, e):
    """Ties, infinite lows and signed zeros among the logits."""
    import mtp_b200
    g = torch.Generator(device=cuda_device).manual_seed(m + e)
    c = layer_case(g, m, e, h, 32, torch.bfloat16, cuda_device)
    logits = torch.randint(-2, 3, (m, e), generator=g, device=cuda_device) * torch.where(
        torch.rand(m, e, generator=g, device=cuda_device) < 0.5, -1.0, 1.0)
    logits[1, 3:] = -float("inf")
    args = (c["w13"], c["s13"], c["w2"], c["s2"], 4)
    w, ids, _ = mtp_b200.topk_softmax(logits, 4)
    given = mtp_b200.moe_layer_w8a8(c["x"], None, *args, topk_weights=w, topk_ids=ids)
    assert torch.equal(mtp_b200.moe_layer_w8a8(c["x"], logits, *args), given)

"""The router's gradient for logits of any finite size: rows masked with the type's lowest value throughout, rows of
large values, large offsets. Against the definition in 64 bits, each output's gradient by itself."""
import pytest
import torch

from test_gpu_route_tokens import BF, F32, HALF, U, definition, logits

pytestmark = pytest.mark.gpu


def rows(value, m, e, dtype):
    """Ordinary rows and, every sixth each: all `value`; `value` but for one of -value; all -value but for two of
    `value`; an ordinary row moved by `value`; `value` with the rest switched off."""
    z, g = logits(m, e, F32, seed=m + e)
    some = torch.randint(0, e, (m,), generator=g, device="cuda")
    at = torch.arange(m, device="cuda")
    kind = at % 6
    z[kind == 1] = value
    z[kind == 2] = value
    z[at[kind == 2], some[kind == 2]] = -value
    z[kind == 3] = -value
    z[at[kind == 3], some[kind == 3]] = value
    z[kind == 3, 0] = value
    z[kind == 4] += value
    z[kind == 5] = value
    z[kind == 5, e // 2:] = -float("inf")
    most = torch.finfo(dtype).max
    return torch.where(z.isinf(), z, z.clamp(-most, most)).to(dtype)


VALUES = [3e4, 1e6, 2.2e9, -3.1e9, 1e10, -1e10, 3e18, 3.3e38, -3.3e38, "highest", "lowest"]


@pytest.mark.parametrize("value", VALUES)
@pytest.mark.parametrize("dtype", [BF, HALF, F32])
@pytest.mark.parametrize("m,e,k", [(7, 20, 4), (300, 64, 6), (60, 300, 8), (40, 1024, 2)])
@pytest.mark.parametrize("renorm", [True, False])
def test_gradient_where_the_logits_are_finite(cuda_device, value, dtype, m, e, k, renorm):
    import mtp_b200
    if isinstance(value, str):
        value = torch.finfo(dtype).max * (1 if value == "highest" else -1)
    z = rows(value, m, e, dtype).requires_grad_()
    z64 = z.detach().double().requires_grad_()
    r = mtp_b200.route_tokens(z, k, renorm)
    want = definition(z64, k, renorm, None)
    assert torch.equal(r.ids.long(), want[1]) and torch.equal(r.counts.long(), want[2])
    # as in the tests of ordinary logits: exponents are below 32 or their probabilities 0
    rel = 256 * U
    assert ((r.weights.double() - want[0]).abs() <= rel * want[0] + 1e-37).all()

    g = torch.Generator(device="cuda").manual_seed(5)
    gw = torch.randn(m, k, generator=g, device="cuda")
    gb, gz = torch.tensor(0.3, device="cuda"), torch.tensor(0.05, device="cuda")
    p, lse = torch.softmax(z64.detach(), -1), torch.logsumexp(z64.detach(), -1, keepdim=True)
    w = want[0].detach()
    pull = 0.3 * e / (k * m * m) * want[2].double()
    of_w = (gw.double().abs() * w).sum(-1, keepdim=True)
    sizes = (torch.zeros_like(p).scatter_(1, want[1], w * (gw.double().abs() + of_w)) + (0 if renorm else p * of_w),
             p * (pull + (pull * p).sum(-1, keepdim=True)), p * (0.1 / m * (1 + lse.abs())))
    info = torch.finfo(dtype)
    # The definition's own error in 64 bits. Renormalised weights give an expert that was not chosen no gradient, but
    # differentiation gives it p_i sum_j p_j d_j with d_j = (g_j - sum g w) / sum p, whose terms cancel:
    # |p_j d_j| <= w_j (|g_j| + of_w), together 2 of_w, after at most e + k + 16 roundings of 2^-53.
    cancelled = 2 * p * of_w * (e + k + 16) * 2.0 ** -53
    # The z loss by its formula: the gradient that torch has for logsumexp is exp(z - lse), and next to 3e18 lse holds
    # nothing of the sum's logarithm in 64 bits either.
    exacts = (*(torch.autograd.grad(o, z64, g.double(), retain_graph=True)[0] for o, g in ((want[0], gw), (want[3], gb))),
              2 * gz.double() / m * lse * p)
    for ours, exact, grad, size in zip((r.weights, r.balance_loss, r.z_loss), exacts, (gw, gb, gz), sizes):
        (got,) = torch.autograd.grad(ours, z, grad, retain_graph=True)
        assert torch.isfinite(got).all()
        bound = 2 * rel * size + info.eps / 2 * exact.abs() + info.smallest_normal * info.eps / 2 + cancelled + 1e-37
        error = (got.double() - exact).abs()
        assert (error <= bound).all(), float((error / bound).max())

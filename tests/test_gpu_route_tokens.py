"""The router with its losses against its definition in 64 bits: weights, ids, counts, losses and the gradient of
the logits, over sizes, types, masks and logits without a finite value."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, HALF, F32, I32 = torch.bfloat16, torch.float16, torch.float32, torch.int32
U = 2.0 ** -24


def definition(z, k, renorm, mask):
    """What route_tokens gives, in 64 bits and differentiable, for logits without NaN."""
    m, e = z.shape
    here = torch.ones(m, dtype=torch.bool, device=z.device) if mask is None else mask
    at = here.nonzero()[:, 0]
    rows = z[at]
    n = max(len(at), 1)
    p = torch.softmax(rows, -1)
    ids = torch.argsort(-rows.detach(), dim=-1, stable=True)[:, :k]
    w = p.gather(1, ids)
    if renorm:
        w = w / w.sum(-1, keepdim=True)
    counts = torch.bincount(ids.flatten(), minlength=e)
    balance = e / (k * n * n) * (counts.double() @ p.sum(0))
    z_loss = torch.logsumexp(rows, -1).square().sum() / n
    weights = torch.zeros(m, k, dtype=z.dtype, device=z.device).index_put((at,), w)
    full = torch.full((m, k), -1, device=z.device)
    full[at] = ids
    return weights, full, counts, balance, z_loss


def logits(m, e, dtype, seed=0, dev="cuda"):
    g = torch.Generator(device=dev).manual_seed(seed)
    z = 1.5 * torch.randn(m, e, generator=g, device=dev) + 0.5 * torch.randn(e, generator=g, device=dev)
    return z.to(dtype), g


def check(z, k, renorm=True, mask=None, grads=True):
    import mtp_b200
    m, e = z.shape
    z = z.detach().requires_grad_(grads)
    z64 = z.detach().double().requires_grad_(grads)
    r = mtp_b200.route_tokens(z, k, renorm, token_mask=mask)
    want = definition(z64, k, renorm, mask)
    assert r.weights.dtype == F32 and r.ids.dtype == I32 and r.counts.dtype == I32
    assert torch.equal(r.ids.long(), want[1]) and torch.equal(r.counts.long(), want[2])
    # z - max is rounded once (|z - max| < 32: 32 u on its exponential), the exponential within 2 units (4 u), a sum
    # of at most 32 + 5 additions of positive terms (37 u), the quotient (u); renormalised: twice that
    rel = 256 * U
    assert (r.weights.double() - want[0]).abs().le(rel * want[0] + 1e-37).all()
    # the loads: as above, and their sum over the tokens (positive terms, a chain of at most m / 8 + 45)
    chain = (m / 8 + 45) * U
    assert abs(float(r.balance_loss.detach()) - float(want[3].detach())) <= (rel + chain) * abs(float(want[3].detach()))
    lse = torch.logsumexp(z64.detach(), -1).abs().max().item() if m else 0.0
    # |error of lse| <= (37 + 4) u of the sum, 2 units of the logarithm (4 u), one rounding (u (lse + 1))
    assert abs(float(r.z_loss.detach()) - float(want[4].detach())) <= 2 * lse * (64 * U * (1 + lse)) + (chain + 4 * U) * lse * lse + 1e-37
    if not grads:
        return
    g = torch.Generator(device=z.device).manual_seed(7)
    gw, gb, gz = torch.randn(m, k, generator=g, device=z.device), torch.tensor(0.3, device=z.device), torch.tensor(0.05, device=z.device)
    (got,) = torch.autograd.grad((r.weights, r.balance_loss, r.z_loss), z, (gw, gb, gz))
    (exact,) = torch.autograd.grad((want[0], want[3], want[4]), z64, (gw.double(), gb.double(), gz.double()))
    assert got.dtype == z.dtype and got.shape == z.shape
    # the terms of the formula with their signs taken off: their errors do not cancel
    here = torch.ones(m, dtype=torch.bool, device=z.device) if mask is None else mask
    n = max(int(here.sum()), 1)
    p = torch.softmax(z64.detach(), -1) * here[:, None]
    pull = 0.3 * e / (k * n * n) * want[2].double()
    ids = want[1].clamp(min=0)
    direct = torch.zeros_like(p).scatter_(1, ids, want[0].detach() * (gw.abs().double() + (gw.double().abs() * want[0].detach()).sum(-1, keepdim=True)))
    size = p * (pull + (pull * p).sum(-1, keepdim=True) + 0.1 / n * (1 + torch.logsumexp(z64.detach(), -1, keepdim=True).abs()))
    if not renorm:  # g stands in the sum over i
        size = size + p * (gw.double().abs() * want[0].detach()).sum(-1, keepdim=True)
    size = torch.where(here[:, None], size + direct, torch.zeros_like(size))
    tiny = torch.finfo(z.dtype).smallest_normal * torch.finfo(z.dtype).eps / 2
    bound = 2 * rel * size + torch.finfo(z.dtype).eps / 2 * exact.abs() + tiny + 1e-37
    assert ((got.double() - exact).abs() <= bound).all(), float(((got.double() - exact).abs() / bound).max())


@pytest.mark.parametrize("m,e,k", [(1, 1, 1), (1, 256, 8), (2, 2, 1), (3, 33, 5), (63, 60, 6), (64, 128, 2), (65, 128, 2),
                                   (300, 257, 8), (513, 31, 31), (129, 1000, 32), (70, 1024, 16), (1000, 64, 4),
                                   (5000, 256, 8), (2400, 512, 1), (20011, 7, 3)])
@pytest.mark.parametrize("renorm", [True, False])
def test_sizes(cuda_device, m, e, k, renorm):
    check(logits(m, e, F32)[0], k, renorm)


@pytest.mark.parametrize("dtype", [BF, HALF, F32])
@pytest.mark.parametrize("share", [0.0, 0.3, 1.0])
@pytest.mark.parametrize("m", [1, 40, 777])
def test_types_and_masks(cuda_device, dtype, share, m):
    z, g = logits(m, 60, dtype)
    mask = torch.rand(m, generator=g, device="cuda") < share
    check(z, 6, True, mask)
    check(z, 6, False, mask)


@pytest.mark.parametrize("m", [5, 500])
def test_rows_that_do_not_count_may_hold_anything(cuda_device, m):
    import mtp_b200
    z, g = logits(m, 40, F32)
    mask = torch.rand(m, generator=g, device="cuda") < 0.5
    dirty = z.clone()
    dirty[~mask] = torch.tensor([float("nan"), float("inf"), -float("inf"), 1e38], device="cuda").repeat(10)
    results = []
    for t in (z, dirty):
        t.requires_grad_()
        r = mtp_b200.route_tokens(t, 4, token_mask=mask)
        (grad,) = torch.autograd.grad(r.weights.square().sum() + r.balance_loss + r.z_loss, t)
        assert not grad[~mask].any()
        results.append((*r, grad))
    for x, y in zip(*results):
        assert torch.equal(x, y)


def test_no_tokens_and_none_that_count(cuda_device):
    import mtp_b200
    for z, mask in ((torch.zeros(0, 8, device="cuda"), None), (torch.randn(9, 8, device="cuda"), torch.zeros(9, dtype=torch.bool, device="cuda")),
                    (torch.randn(900, 8, device="cuda"), torch.zeros(900, dtype=torch.bool, device="cuda"))):
        z.requires_grad_()
        r = mtp_b200.route_tokens(z, 2, token_mask=mask)
        assert r.counts.tolist() == [0] * 8 and float(r.balance_loss) == 0 and float(r.z_loss) == 0
        assert (r.ids == -1).all() and not r.weights.any()
        (grad,) = torch.autograd.grad(r.weights.sum() + r.balance_loss + r.z_loss, z)
        assert grad.shape == z.shape and not grad.any()


@pytest.mark.parametrize("m", [8, 200])
def test_experts_that_are_switched_off(cuda_device, m):
    """Logits of -inf: weight and gradient 0; they are chosen only when nothing else is left."""
    import mtp_b200
    z, _ = logits(m, 24, F32)
    z[:, 5] = -float("inf")
    z[: m // 2, 12:] = -float("inf")
    check(z, 8)
    z[0, 3:] = -float("inf")  # three experts left for eight choices
    z.requires_grad_()
    r = mtp_b200.route_tokens(z, 8)
    assert sorted(r.ids[0, :3].tolist()) == [0, 1, 2] and r.ids[0, 3:].tolist() == [3, 4, 5, 6, 7]
    assert not r.weights[0, 3:].any() and abs(float(r.weights[0].sum()) - 1) <= 8 * U
    (grad,) = torch.autograd.grad(r.weights.square().sum() + r.balance_loss + r.z_loss, z)
    assert torch.isfinite(grad).all() and not grad[0, 3:].any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("m", [3, 300])
def test_bad_logits_are_not_lost(cuda_device, bad, m):
    import mtp_b200
    z, _ = logits(m, 20, F32)
    z[1, 7] = bad
    z[2] = bad
    r = mtp_b200.route_tokens(z, 4)
    assert torch.isnan(r.weights[1:3]).all() and torch.isfinite(r.weights[0]).all()
    assert torch.isnan(r.balance_loss) and torch.isnan(r.z_loss)
    for t in range(m):
        assert len(set(r.ids[t].tolist())) == 4 and 0 <= r.ids[t].min() and r.ids[t].max() < 20
    assert int(r.counts.sum()) == 4 * m


@pytest.mark.parametrize("dtype", [BF, F32])
def test_ties_go_to_the_lowest_expert(cuda_device, dtype):
    import mtp_b200
    z = torch.zeros(70, 90, dtype=dtype, device="cuda")
    z[:, 1::2] = -0.0
    assert mtp_b200.route_tokens(z, 5).ids.tolist() == [[0, 1, 2, 3, 4]] * 70
    z[:, [80, 40, 33]] = 1
    assert mtp_b200.route_tokens(z, 5).ids.tolist() == [[33, 40, 80, 0, 1]] * 70


def test_as_topk_softmax(cuda_device):
    import mtp_b200
    for e, k in ((60, 6), (256, 8), (1000, 10)):
        z, _ = logits(333, e, F32)
        w, ids, _ = mtp_b200.topk_softmax(z, k)
        r = mtp_b200.route_tokens(z, k)
        assert torch.equal(r.ids, ids) and torch.equal(r.weights, w)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_of_a_wider_tensor(cuda_device, dtype):
    import mtp_b200
    wide, _ = logits(100, 77, dtype)
    z = wide[:, 3:64].requires_grad_()
    r = mtp_b200.route_tokens(z, 3)
    (grad,) = torch.autograd.grad(r.weights[:, 0].sum() + r.balance_loss, z)
    c = z.detach().clone().requires_grad_()
    q = mtp_b200.route_tokens(c, 3)
    (want,) = torch.autograd.grad(q.weights[:, 0].sum() + q.balance_loss, c)
    for x, y in zip((*r, grad), (*q, want)):
        assert torch.equal(x, y)


def test_each_gradient_alone_and_their_sum(cuda_device):
    import mtp_b200
    z, _ = logits(150, 48, F32)
    z.requires_grad_()
    r = mtp_b200.route_tokens(z, 4)
    gw = torch.randn(150, 4, device="cuda")
    one = torch.ones((), device="cuda")
    parts = [torch.autograd.grad(o, z, g, retain_graph=True)[0] for o, g in ((r.weights, gw), (r.balance_loss, one), (r.z_loss, one))]
    (whole,) = torch.autograd.grad((r.weights, r.balance_loss, r.z_loss), z, (gw, one, one), retain_graph=True)
    assert all(p.any() for p in parts)
    # four roundings of sums no larger than the parts' sizes
    assert ((whole - sum(parts)).abs() <= 16 * U * sum(p.abs() for p in parts) + 1e-9).all()
    # a gradient that is not contiguous
    (got,) = torch.autograd.grad(r.weights, z, gw.t().contiguous().t())
    assert torch.equal(got, parts[0])


def test_gradient_against_differences(cuda_device):
    """Central differences of the definition in 64 bits along random directions."""
    import mtp_b200
    z, g = logits(40, 24, F32)
    z.requires_grad_()
    r = mtp_b200.route_tokens(z, 3)
    gw = torch.randn(40, 3, generator=g, device="cuda")

    def loss(t):
        # choices and counts are constants of the gradient
        p = torch.softmax(t, -1)
        w = p.gather(1, r.ids.long())
        w = w / w.sum(-1, keepdim=True)
        return (w * gw).sum() + 0.5 * 24 / (3 * 1600) * (r.counts.double() @ p.sum(0)) + 0.1 * torch.logsumexp(t, -1).square().mean()

    (grad,) = torch.autograd.grad((r.weights * gw).sum() + 0.5 * r.balance_loss + 0.1 * r.z_loss, z)
    for _ in range(5):
        d = torch.randn(40, 24, generator=g, device="cuda", dtype=torch.float64)
        h = 1e-5
        with torch.no_grad():
            slope = (loss(z.double() + h * d) - loss(z.double() - h * d)) / (2 * h)
        # h^2 of the third derivative (below 1e-8), and the gradient's 2^-15 of its terms
        assert abs(float((grad.double() * d).sum() - slope)) <= 2.0 ** -15 * float((grad.double() * d).abs().sum()) + 1e-7


def test_same_bits_again(cuda_device):
    import mtp_b200
    z, _ = logits(9000, 256, F32)
    z.requires_grad_()

    def results():
        r = mtp_b200.route_tokens(z, 8)
        return (*r, *torch.autograd.grad(r.weights.square().sum() + r.balance_loss + r.z_loss, z))

    first = results()
    for _ in range(3):
        for x, y in zip(results(), first):
            assert torch.equal(x, y)


def test_offsets_past_32_bits(cuda_device):
    """More than 2^31 logits: the last tokens are as in a call of their own."""
    import mtp_b200
    m, e = 2_150_000, 1000
    z = torch.zeros(m, e, dtype=BF, device="cuda")
    tail, _ = logits(300, e, BF)
    z[-300:] = tail
    mask = torch.zeros(m, dtype=torch.bool, device="cuda")
    mask[-300:] = True
    results = []
    for rows, counted in ((z, mask), (tail, None)):
        rows.requires_grad_()
        r = mtp_b200.route_tokens(rows, 6, token_mask=counted)
        (grad,) = torch.autograd.grad(r.weights.square().sum() + r.balance_loss + r.z_loss, rows)
        results.append((r.weights[-300:], r.ids[-300:], r.counts, grad[-300:].clone()))
        assert rows is tail or not grad[:-300].any()
        del grad
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
    assert torch.equal(results[0][2], results[1][2]) and torch.equal(results[0][3], results[1][3])

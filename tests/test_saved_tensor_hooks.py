"""Saved-tensor hooks (offloading, compression) give a backward pass other tensors than the forward pass saved: dense
where a slice of wider rows was saved, in another memory order, or wrong ones. What the C entries get has to be that
tensor's layout. On the CPU with recorded entries; the GPU tests compare gradients with and without hooks."""
import pytest
import torch
import torch.utils.checkpoint

import mtp_b200
from mtp_b200 import training, w8a8

I32 = torch.int32


@pytest.fixture
def entries(built_lib, monkeypatch):
    """Host tensors are taken as a GPU's; the C entries only record their arguments."""
    calls = {}
    for module, names in ((training, ("route", "route_backward", "norm", "norm_backward", "embed", "embed_backward")),
                          (w8a8, ("sort", "unsort", "unsort_backward"))):
        for name in names:
            monkeypatch.setattr(module, f"_{name}_entry", lambda *args, name=name: calls.__setitem__(name, args))
        monkeypatch.setattr(module, "_tensor", lambda *args, **kwargs: None)
        monkeypatch.setattr(module, "_current_device", lambda: -1)
        monkeypatch.setattr(module, "_stream", lambda device: 0)
    return calls


class Hooks(torch.autograd.graph.saved_tensors_hooks):
    """Hooks whose unpacked tensors are change(saved), kept in ``given`` by shape."""

    def __init__(self, change):
        self.given = []

        def unpack(t):
            t = change(t)
            self.given.append(t)
            return t

        super().__init__(lambda t: t, unpack)

    def at(self, pointer):
        return next((t for t in self.given if t.data_ptr() == pointer), None)


def dense(t):
    return t.clone(memory_format=torch.contiguous_format)


def wider(t):
    """The same values as rows of a wider tensor."""
    if t.ndim != 2 or not t.is_floating_point():
        return dense(t)
    return torch.nn.functional.pad(t, (0, 5))[:, :t.shape[1]]


def columns_first(t):
    return t.t().contiguous().t() if t.ndim == 2 else dense(t)


def _logits(m=20, e=9, wide=32):
    return torch.randn(m, wide)[:, 3:3 + e].requires_grad_()


@pytest.mark.parametrize("change,stride", [(dense, 9), (wider, 14), (columns_first, 9)])
def test_route_takes_the_stride_of_the_unpacked_logits(entries, change, stride):
    z = _logits()
    hooks = Hooks(change)
    with hooks:
        r = mtp_b200.route_tokens(z, 2, token_mask=torch.ones(20, dtype=torch.bool))
        r.weights.sum().backward()
    assert entries["route"][:2] == (z.data_ptr(), 32)
    pointer, got = entries["route_backward"][:2]
    assert got == stride
    given = hooks.at(pointer)
    assert given is None if change is columns_first else given.stride(0) == stride


@pytest.mark.parametrize("change,stride", [(dense, 9), (wider, 14), (columns_first, 9)])
def test_layer_norm_takes_the_stride_of_the_unpacked_rows(entries, change, stride):
    x = _logits()
    w = torch.ones(9, requires_grad=True)
    hooks = Hooks(change)
    with hooks:
        mtp_b200.layer_norm(x, w).sum().backward()
    assert entries["norm"][:2] == (x.data_ptr(), 32)
    _, pointer, got = entries["norm_backward"][:3]
    assert got == stride
    given = hooks.at(pointer)
    assert given is None if change is columns_first else given.stride(0) == stride


def test_layer_norm_of_more_dimensions(entries):
    x = torch.randn(2, 5, 7, requires_grad=True)
    with Hooks(lambda t: t.transpose(0, 1).contiguous().transpose(0, 1) if t.ndim == 3 else t):
        mtp_b200.layer_norm(x).sum().backward()
    args = entries["norm_backward"]
    assert args[2] == 7 and args[4:6] == (10, 7)


def test_without_hooks_slices_stay_slices(entries):
    z, x = _logits(), _logits()
    (mtp_b200.route_tokens(z, 2).weights.sum() + mtp_b200.layer_norm(x).sum()).backward()
    assert entries["route_backward"][:2] == (z.data_ptr(), 32) and entries["norm_backward"][1:3] == (x.data_ptr(), 32)


WRONG = {
    "shape": lambda t: t[:-1],
    "size": lambda t: torch.cat([t, t]),
    "type": lambda t: t.double() if t.is_floating_point() else t.to(torch.int16),
}


@pytest.mark.parametrize("wrong", WRONG.values(), ids=WRONG)
@pytest.mark.parametrize("which", range(4))
def test_route_refuses_other_tensors(entries, wrong, which):
    z, seen = _logits(), []
    with Hooks(lambda t: (seen.append(t), wrong(t) if len(seen) == which + 1 else t)[1]):
        r = mtp_b200.route_tokens(z, 2, token_mask=torch.ones(20, dtype=torch.bool))
        with pytest.raises(RuntimeError, match="saved"):
            r.weights.sum().backward()
    assert len(seen) == 4 and "route_backward" not in entries


@pytest.mark.parametrize("wrong", WRONG.values(), ids=WRONG)
@pytest.mark.parametrize("which", range(3))
def test_layer_norm_refuses_other_tensors(entries, wrong, which):
    x, w, seen = _logits(), torch.ones(9, requires_grad=True), []
    with Hooks(lambda t: (seen.append(t), wrong(t) if len(seen) == which + 1 else t)[1]):
        y = mtp_b200.layer_norm(x, w)
        with pytest.raises(RuntimeError, match="saved"):
            y.sum().backward()
    assert len(seen) == 3 and "norm_backward" not in entries


@pytest.mark.parametrize("wrong", WRONG.values(), ids=WRONG)
def test_embedding_refuses_other_ids(entries, wrong):
    table = torch.randn(8, 5, requires_grad=True)
    with Hooks(wrong):
        out = mtp_b200.embed_tokens(torch.arange(6, dtype=I32), table)
        with pytest.raises(RuntimeError, match="saved"):
            out.sum().backward()
    assert "embed_backward" not in entries


def test_a_tensor_left_on_another_device_is_refused(entries, monkeypatch):
    """As where a hook forgets the way back to the GPU."""
    x = _logits()
    with Hooks(lambda t: t.to("meta") if t.ndim == 2 and t.shape[1] == 9 else t):
        y = mtp_b200.layer_norm(x)
        with pytest.raises(RuntimeError, match="saved"):
            y.sum().backward()
        r = mtp_b200.route_tokens(x, 2)
        with pytest.raises(RuntimeError, match="saved"):
            r.weights.sum().backward()
    assert "norm_backward" not in entries and "route_backward" not in entries


def _pairs():
    rows, weights = torch.randn(6, 5, requires_grad=True), torch.rand(3, 2, requires_grad=True)
    return rows, torch.tensor([[0, 3], [4, 1], [2, 5]], dtype=I32), weights


def test_unsort_takes_tensors_in_row_order(entries):
    rows, positions, weights = _pairs()
    hooks = Hooks(columns_first)
    with hooks:
        mtp_b200.unsort_tokens(rows, positions, weights).sum().backward()
    _, at_rows, num_rows, _, at_positions, at_weights = entries["unsort_backward"][:6]
    assert num_rows == 6 and len(hooks.given) == 3
    assert not any(hooks.at(p) is not None for p in (at_rows, at_positions, at_weights))  # copies in row order


def test_sort_takes_positions_in_row_order(entries):
    x, hooks = torch.randn(3, 5, requires_grad=True), Hooks(columns_first)
    with hooks:
        mtp_b200.sort_tokens(x, torch.zeros(3, 2, dtype=I32), 4).rows.sum().backward()
    assert len(hooks.given) == 1 and hooks.at(entries["unsort"][3]) is None


def test_sort_and_unsort_without_hooks_make_no_copies(entries):
    rows, positions, weights = _pairs()
    mtp_b200.unsort_tokens(rows, positions, weights).sum().backward()
    args = entries["unsort_backward"]
    assert (args[1], args[4], args[5]) == (rows.data_ptr(), positions.data_ptr(), weights.data_ptr())


@pytest.mark.parametrize("wrong", WRONG.values(), ids=WRONG)
@pytest.mark.parametrize("which", range(3))
def test_unsort_refuses_other_tensors(entries, wrong, which):
    (rows, positions, weights), seen = _pairs(), []
    with Hooks(lambda t: (seen.append(t), wrong(t) if len(seen) == which + 1 else t)[1]):
        y = mtp_b200.unsort_tokens(rows, positions, weights)
        with pytest.raises(RuntimeError, match="saved"):
            y.sum().backward()
    assert len(seen) == 3 and "unsort_backward" not in entries


@pytest.mark.parametrize("wrong", WRONG.values(), ids=WRONG)
def test_sort_refuses_other_positions(entries, wrong):
    x = torch.randn(3, 5, requires_grad=True)
    with Hooks(wrong):
        r = mtp_b200.sort_tokens(x, torch.zeros(3, 2, dtype=I32), 4)
        with pytest.raises(RuntimeError, match="saved"):
            r.rows.sum().backward()
    assert "unsort" not in entries


@pytest.mark.gpu
class TestOnTheGpu:
    @pytest.fixture(params=["on the host", "pinned", "dense", "wider", "columns first", "checkpoint"])
    def around(self, request, cuda_device):
        """call(fn, *args): fn with hooks around it."""
        if request.param == "checkpoint":
            return lambda fn, *args: torch.utils.checkpoint.checkpoint(fn, *args, use_reentrant=False)
        hooks = {"on the host": torch.autograd.graph.save_on_cpu, "pinned": lambda: torch.autograd.graph.save_on_cpu(pin_memory=True),
                 "dense": lambda: Hooks(dense), "wider": lambda: Hooks(wider), "columns first": lambda: Hooks(columns_first)}[request.param]

        def call(fn, *args):
            with hooks():
                return fn(*args)

        return call

    @pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
    @pytest.mark.parametrize("m", [5, 700])
    def test_route(self, around, m, dtype):
        g = torch.Generator(device="cuda").manual_seed(m)
        wide = torch.randn(m, 77, generator=g, device="cuda").to(dtype)
        mask = torch.rand(m, generator=g, device="cuda") < 0.8
        z = wide[:, 3:64].requires_grad_()
        gw = torch.randn(m, 3, generator=g, device="cuda")

        def loss(t):
            r = mtp_b200.route_tokens(t, 3, token_mask=mask)
            return (r.weights * gw).sum() + r.balance_loss + r.z_loss

        (want,) = torch.autograd.grad(loss(z), z)
        (got,) = torch.autograd.grad(around(loss, z), z)
        assert torch.equal(got, want)

    @pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
    @pytest.mark.parametrize("m,h,start,wide", [(5, 61, 3, 77), (700, 61, 3, 77), (700, 512, 0, 1024), (20, 512, 8, 640)])
    def test_layer_norm(self, around, m, h, start, wide, dtype):
        g = torch.Generator(device="cuda").manual_seed(m)
        x = torch.randn(m, wide, generator=g, device="cuda").to(dtype)[:, start:start + h].requires_grad_()
        w, b = (torch.randn(h, generator=g, device="cuda", requires_grad=True) for _ in range(2))
        gy = torch.randn(m, h, generator=g, device="cuda").to(dtype)
        want = torch.autograd.grad(mtp_b200.layer_norm(x, w, b), (x, w, b), gy)
        got = torch.autograd.grad(around(mtp_b200.layer_norm, x, w, b), (x, w, b), gy)
        # Another layout of the rows may put their values into another order: on either side at most (h / 32 + 40) u of a
        # row's sums and (m / 32 + 64) u of a column's, of the sums of absolute values, and four roundings of the last
        # step; then half a step of the rows' type.
        u, rel = 2.0 ** -24, torch.finfo(dtype).eps / 2
        x64, wg = x.detach().double(), gy.double() * w.detach().double()
        rstd = 1 / (x64.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt()
        xhat = (x64 - x64.mean(-1, keepdim=True)) * rstd
        mean = lambda t: t.abs().mean(-1, keepdim=True)
        size = rstd * (wg.abs() + mean(wg) + xhat.abs() * mean(wg * xhat))
        bounds = (2 * (h / 32 + 44) * u * size + 2 * rel * want[0].double().abs(),
                  2 * (m / 32 + 64) * u * (gy.double() * xhat).abs().sum(0), 2 * (m / 32 + 64) * u * gy.double().abs().sum(0))
        for p, q, bound in zip(got, want, bounds):
            assert ((p.double() - q.double()).abs() <= bound * (1 + 2 * rel)).all()

    def test_embedding(self, around):
        g = torch.Generator(device="cuda").manual_seed(1)
        table = torch.randn(50, 24, generator=g, device="cuda", requires_grad=True)
        ids = torch.randint(-1, 50, (20, 10), generator=g, device="cuda")
        gy = torch.randn(20, 10, 24, generator=g, device="cuda")
        (want,) = torch.autograd.grad(mtp_b200.embed_tokens(ids, table), table, gy)
        (got,) = torch.autograd.grad(around(lambda t: mtp_b200.embed_tokens(ids, t), table), table, gy)
        assert torch.equal(got, want)

    def test_sort_and_unsort(self, around):
        g = torch.Generator(device="cuda").manual_seed(2)
        x = torch.randn(90, 40, generator=g, device="cuda", requires_grad=True)
        w = torch.rand(90, 3, generator=g, device="cuda", requires_grad=True)
        ids = torch.randint(-1, 7, (90, 3), generator=g, device="cuda", dtype=I32)
        gy = torch.randn(90, 40, generator=g, device="cuda")

        def there_and_back(x, w):
            r = mtp_b200.sort_tokens(x, ids, 7)
            return mtp_b200.unsort_tokens(r.rows * 2, r.positions, w)

        want = torch.autograd.grad(there_and_back(x, w), (x, w), gy)
        got = torch.autograd.grad(around(there_and_back, x, w), (x, w), gy)
        assert all(torch.equal(p, q) for p, q in zip(got, want))

"""What the operators of a training step refuse, in Python before a launch and at the C entries with a status; and
the device that is current at their launches. CPU only, but for the class at the end."""
import contextlib
import ctypes as C

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mtp_b200
from mtp_b200 import training

I32, I64, BF, F32 = torch.int32, torch.int64, torch.bfloat16, torch.float32
LIMIT = 2 ** 31 - 65536


@pytest.mark.parametrize("name,args", [
    ("route_tokens", (torch.zeros(2, 4), 2)),
    ("layer_norm", (torch.zeros(2, 4),)),
    ("embed_tokens", (torch.zeros(2, dtype=I32), torch.zeros(3, 4))),
])
def test_host_tensors_are_refused(built_lib, name, args):
    with pytest.raises(ValueError, match="CUDA"):
        getattr(mtp_b200, name)(*args)
    with pytest.raises(TypeError):
        getattr(mtp_b200, name)([1.0], *args[1:])


@pytest.fixture
def c(built_lib):
    from mtp_b200 import _lib
    lib = _lib.load()
    buf = (C.c_uint8 * 4096)()
    p = C.addressof(buf) + (-C.addressof(buf)) % 256
    big = 1 << 40

    def route(z=p, stride=8, dt=0, m=2, e=8, k=2, mask=None, w=p, ids=p, counts=p, bal=p, zl=p, pull=p, ws=p, size=big):
        return lib.mtp_route_tokens(z, stride, dt, m, e, k, 1, mask, w, ids, counts, bal, zl, pull, ws, size, None)

    def route_back(z=p, stride=8, dt=0, m=2, e=8, k=2, ids=p, pull=p, gw=p, gb=p, gz=p, g=p):
        return lib.mtp_route_tokens_backward(z, stride, dt, m, e, k, 1, None, ids, pull, gw, gb, gz, g, None)

    def route_size(m=2, e=8):
        return lib.mtp_route_tokens_workspace_size(m, e, C.byref(C.c_int64()))

    def norm(x=p, stride=8, dt=0, m=2, h=8, w=p, b=p, pt=2, eps=1e-5, y=p, stats=p):
        return lib.mtp_layer_norm(x, stride, dt, m, h, w, b, pt, eps, y, stats, None)

    def norm_back(g=p, x=p, stride=8, dt=0, m=2, h=8, w=p, pt=2, stats=p, gx=p, gw=p, gb=p, ws=p, size=big):
        return lib.mtp_layer_norm_backward(g, x, stride, dt, m, h, w, pt, stats, gx, gw, gb, ws, size, None)

    def norm_size(m=2, h=8):
        return lib.mtp_layer_norm_backward_workspace_size(m, h, C.byref(C.c_int64()))

    def embed(ids=p, width=4, n=2, table=p, dt=0, v=4, h=8, out=p):
        return lib.mtp_embed_tokens(ids, width, n, table, dt, v, h, 1.0, out, None)

    def embed_back(ids=p, width=4, n=2, g=p, dt=0, v=4, h=8, gt=p, ws=p, size=big):
        return lib.mtp_embed_tokens_backward(ids, width, n, g, dt, v, h, 1.0, gt, ws, size, None)

    def embed_size(n=2, h=8, dt=0):
        return lib.mtp_embed_tokens_backward_workspace_size(n, h, dt, C.byref(C.c_int64()))

    return dict(locals())


LAST = 2 ** 31 - 1
REFUSED = [
    ("route", 1, [dict(z=None), dict(w=None), dict(ids=None), dict(counts=None), dict(bal=None), dict(zl=None), dict(m=500, ws=None)]),
    ("route", 2, [dict(m=-1), dict(e=0), dict(e=1025, stride=1025), dict(k=0), dict(k=9), dict(e=64, stride=64, k=33), dict(stride=7),
                  dict(m=LIMIT + 1, k=1), dict(m=LAST, k=1), dict(m=2 ** 30, k=2)]),
    ("route", 3, [dict(z="odd"), dict(ws="odd", m=500)]),
    ("route", 4, [dict(m=500, size=64)]),
    ("route", 9, [dict(dt=3), dict(dt=-1)]),
    ("route_size", 2, [dict(m=-1), dict(m=LAST), dict(e=0), dict(e=1025)]),
    ("route_back", 1, [dict(z=None), dict(g=None), dict(ids=None), dict(pull=None), dict(pull=None, gb=None)]),
    ("route_back", 2, [dict(m=-1), dict(e=1025, stride=1025), dict(k=9), dict(stride=7), dict(m=LAST, k=1)]),
    ("route_back", 3, [dict(z="odd"), dict(g="odd")]),
    ("route_back", 9, [dict(dt=3)]),
    ("route_back", 0, [dict(m=0, z=None, g=None, ids=None, pull=None)]),
    ("norm", 1, [dict(x=None), dict(y=None)]),
    ("norm", 2, [dict(m=-1), dict(h=0), dict(stride=7), dict(m=LIMIT + 1), dict(h=LIMIT + 1, stride=LAST), dict(m=LAST), dict(h=LAST, stride=LAST)]),
    ("norm", 3, [dict(x="odd"), dict(y="odd"), dict(w="odd"), dict(b="odd"), dict(stats="odd")]),
    ("norm", 9, [dict(dt=3), dict(pt=1), dict(dt=2, pt=0), dict(eps=-1.0), dict(eps=float("nan"))]),
    ("norm", 0, [dict(m=0, x=None, y=None)]),
    ("norm_back", 1, [dict(g=None), dict(x=None), dict(stats=None), dict(ws=None)]),
    ("norm_back", 2, [dict(m=-1), dict(h=0), dict(stride=7), dict(m=LAST), dict(h=LAST, stride=LAST)]),
    ("norm_back", 3, [dict(g="odd"), dict(x="odd"), dict(gx="odd"), dict(gw="odd"), dict(gb="odd"), dict(w="odd"), dict(ws="odd"), dict(stats="odd")]),
    ("norm_back", 4, [dict(size=1)]),
    ("norm_back", 9, [dict(dt=3), dict(pt=1)]),
    ("norm_back", 0, [dict(gx=None, gw=None, gb=None)]),
    ("norm_size", 2, [dict(m=-1), dict(m=LAST), dict(h=0), dict(h=LAST)]),
    ("embed", 1, [dict(ids=None), dict(table=None), dict(out=None)]),
    ("embed", 2, [dict(n=-1), dict(v=0), dict(h=0), dict(n=LAST), dict(v=LAST), dict(h=LAST), dict(n=LIMIT + 1), dict(h=LIMIT + 1)]),
    ("embed", 3, [dict(ids="odd"), dict(table="odd"), dict(out="odd"), dict(ids="four", width=8)]),
    ("embed", 9, [dict(dt=3), dict(width=2)]),
    ("embed", 0, [dict(n=0, ids=None, table=None, out=None)]),
    ("embed_back", 1, [dict(ids=None), dict(g=None), dict(gt=None), dict(ws=None)]),
    ("embed_back", 2, [dict(n=-1), dict(v=0), dict(h=0), dict(n=LAST), dict(v=LAST), dict(h=LAST)]),
    ("embed_back", 3, [dict(ids="odd"), dict(g="odd"), dict(gt="odd"), dict(ws="odd")]),
    ("embed_back", 4, [dict(size=16)]),
    ("embed_back", 9, [dict(dt=3), dict(width=1)]),
    ("embed_size", 2, [dict(n=-1), dict(n=LAST), dict(h=0), dict(h=LAST)]),
    ("embed_size", 9, [dict(dt=3)]),
]


@pytest.mark.parametrize("entry,status,calls", REFUSED, ids=lambda x: x if isinstance(x, (str, int)) else "")
def test_c_entries(c, entry, status, calls):
    for call in calls:
        got = c[entry](**{n: c["p"] + {"odd": 1, "four": 4}[v] if isinstance(v, str) else v for n, v in call.items()})
        assert got == status, (call, got)


def test_size_queries_take_the_largest(c):
    lib, out = c["lib"], C.c_int64()
    assert lib.mtp_route_tokens_workspace_size(LIMIT, 1024, C.byref(out)) == 0 and 0 < out.value < 1 << 24
    assert lib.mtp_route_tokens_workspace_size(1, 1024, C.byref(out)) == 0 and out.value == 0
    assert lib.mtp_layer_norm_backward_workspace_size(LIMIT, LIMIT - 1, C.byref(out)) == 0 and out.value >= 8 * (LIMIT - 1)
    assert lib.mtp_embed_tokens_backward_workspace_size(LIMIT - 1, LIMIT - 1, 2, C.byref(out)) == 0 and out.value > 0
    for call in ((lib.mtp_route_tokens_workspace_size, 2, 8), (lib.mtp_layer_norm_backward_workspace_size, 2, 8),
                 (lib.mtp_embed_tokens_backward_workspace_size, 2, 8, 0)):
        assert call[0](*call[1:], None) == 1


class Entries:
    """Stands for the C entries: what was called, and which device was current then."""

    def __init__(self, monkeypatch, current):
        self.current, self.calls = current, []
        for name in ("route", "route_backward", "norm", "norm_backward", "embed", "embed_backward"):
            monkeypatch.setattr(training, f"_{name}_entry", lambda *args, name=name: self.calls.append((name, self.current, args[-1])))
        monkeypatch.setattr(training, "_current_device", lambda: self.current)
        monkeypatch.setattr(training, "_stream", lambda device: 1000 + device)
        monkeypatch.setattr(torch.cuda, "device", self.device)
        monkeypatch.setattr(torch.cuda, "is_available", lambda: False)  # fake tensors of a GPU that is not there

    @contextlib.contextmanager
    def device(self, index):
        before, self.current = self.current, index
        try:
            yield
        finally:
            self.current = before


@pytest.mark.filterwarnings("ignore:Accessing the data pointer of FakeTensor")
@pytest.mark.parametrize("index,current", [(1, 0), (0, 0), (0, 3)])
def test_the_tensors_device_is_current_at_the_launch(built_lib, monkeypatch, index, current):
    entries = Entries(monkeypatch, current)
    with FakeTensorMode():
        z = lambda *shape, dtype=F32: torch.empty(*shape, dtype=dtype, device=f"cuda:{index}")
        for name, call in [
            ("route", lambda: mtp_b200.route_tokens(z(4, 8), 2)),
            ("route_backward", lambda: training._route_backward(z(4, 8), 8, 2, True, None, z(4, 2, dtype=I32), z(9), z(4, 2), None, None)),
            ("norm", lambda: mtp_b200.layer_norm(z(4, 8), z(8), z(8))),
            ("norm_backward", lambda: training._norm_backward(z(4, 8), z(4, 8), (4, 8), z(8), z(4, 2), F32, True, True, True)),
            ("embed", lambda: mtp_b200.embed_tokens(z(4, dtype=I32), z(5, 8))),
            ("embed_backward", lambda: training._embed_backward(z(4, dtype=I32), z(4, 8), 5, 1.0)),
        ]:
            entries.calls.clear()
            call()
            assert entries.calls == [(name, index, 1000 + index)]
            assert entries.current == current


@pytest.mark.filterwarnings("ignore:Accessing the data pointer of FakeTensor")
@pytest.mark.parametrize("n", [LIMIT + 1, 2 ** 31, 2 ** 32 + 8])
def test_python_refuses_what_32_bits_do_not_index(built_lib, monkeypatch, n):
    Entries(monkeypatch, 0)
    taken = []
    with FakeTensorMode():
        z = lambda *shape, dtype=F32: torch.empty(*shape, dtype=dtype, device="cuda:0")
        for name, call in {
            "pairs": lambda: mtp_b200.route_tokens(z(n, 2, dtype=BF), 1),
            "rows": lambda: mtp_b200.layer_norm(z(n, 1)),
            "columns": lambda: mtp_b200.layer_norm(z(2, n, dtype=BF)),
            "ids": lambda: mtp_b200.embed_tokens(z(n, dtype=I32), z(2, 2)),
            "table rows": lambda: mtp_b200.embed_tokens(z(2, dtype=I32), z(n, 1)),
            "table columns": lambda: mtp_b200.embed_tokens(z(2, dtype=I32), z(1, n, dtype=BF)),
        }.items():
            try:
                call()
                taken.append(name)
            except ValueError as e:
                assert "supported" in str(e), name
    assert not taken


class TestOnTheGpu:
    pytestmark = pytest.mark.gpu

    def test_shapes_types_and_layouts(self, cuda_device):
        z = lambda *s, dtype=F32: torch.zeros(*s, dtype=dtype, device=cuda_device)
        x, ids = z(4, 8), z(4, dtype=I32)
        bad = [
            ("route_tokens", (x.double(), 2), {}), ("route_tokens", (x, 0), {}), ("route_tokens", (x, 9), {}), ("route_tokens", (z(4), 1), {}),
            ("route_tokens", (z(4, 0), 1), {}), ("route_tokens", (z(2, 1025), 1), {}), ("route_tokens", (z(2, 64), 33), {}),
            ("route_tokens", (x.t(), 2), {}), ("route_tokens", (x[:1].expand(4, 8), 2), {}),
            ("route_tokens", (x, 2), dict(token_mask=z(3, dtype=torch.bool))), ("route_tokens", (x, 2), dict(token_mask=z(4, dtype=torch.uint8))),
            ("route_tokens", (x, 2), dict(token_mask=z(8, dtype=torch.bool)[::2])),
            ("route_tokens", (x, 2), dict(token_mask=torch.ones(4, dtype=torch.bool))),
            ("layer_norm", (x.double(),), {}), ("layer_norm", (z(()),), {}), ("layer_norm", (z(4, 0),), {}), ("layer_norm", (x.t(),), {}),
            ("layer_norm", (z(2, 2, 8).transpose(0, 1),), {}), ("layer_norm", (x, z(7)), {}), ("layer_norm", (x, z(8), z(9)), {}),
            ("layer_norm", (x, z(8, dtype=BF)), {}), ("layer_norm", (x.to(BF), z(8, dtype=torch.float16)), {}),
            ("layer_norm", (x.to(BF), z(8, dtype=BF), z(8)), {}), ("layer_norm", (x, z(16)[::2]), {}), ("layer_norm", (x, torch.zeros(8)), {}),
            ("layer_norm", (x,), dict(eps=-1.0)), ("layer_norm", (x,), dict(eps=float("nan"))), ("layer_norm", (x,), dict(eps=float("inf"))),
            ("embed_tokens", (ids.float(), x), {}), ("embed_tokens", (ids.to(torch.int16), x), {}), ("embed_tokens", (ids, z(4)), {}),
            ("embed_tokens", (ids, x.double()), {}), ("embed_tokens", (ids, x.t()), {}), ("embed_tokens", (ids, z(0, 8)), {}),
            ("embed_tokens", (ids, z(4, 0)), {}), ("embed_tokens", (ids[::2], x), {}), ("embed_tokens", (ids.cpu(), x), {}),
            ("embed_tokens", (ids, x), dict(scale=float("inf"))), ("embed_tokens", (ids, x), dict(scale=torch.ones((), device=cuda_device))),
        ]
        for name, args, kw in bad:
            with pytest.raises(ValueError):
                getattr(mtp_b200, name)(*args, **kw)
        torch.cuda.synchronize()

    @pytest.mark.parametrize("grad_enabled", [True, False])
    def test_forward_mode_raises(self, cuda_device, grad_enabled):
        from torch.autograd import forward_ad
        x, w, ids = torch.randn(6, 8, device=cuda_device), torch.ones(8, device=cuda_device), torch.zeros(3, dtype=I32, device=cuda_device)
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        with forward_ad.dual_level(), torch.set_grad_enabled(grad_enabled):
            for call in (lambda: mtp_b200.route_tokens(dual(x), 2), lambda: mtp_b200.layer_norm(dual(x)), lambda: mtp_b200.layer_norm(x, dual(w)),
                         lambda: mtp_b200.layer_norm(x, w, dual(w)), lambda: mtp_b200.embed_tokens(ids, dual(x))):
                with pytest.raises(RuntimeError, match="jvp|forward mode"):
                    call()

    def test_second_derivatives_raise(self, cuda_device):
        x = torch.randn(6, 8, device=cuda_device, requires_grad=True)
        ids = torch.zeros(3, dtype=I32, device=cuda_device)
        for out in (mtp_b200.route_tokens(x, 2).weights, mtp_b200.layer_norm(x), mtp_b200.embed_tokens(ids, x)):
            (g,) = torch.autograd.grad(out.square().sum(), x, create_graph=True)
            with pytest.raises(RuntimeError):
                torch.autograd.grad(g.sum(), x)

    def test_no_grad_records_nothing(self, cuda_device):
        x = torch.randn(6, 8, device=cuda_device, requires_grad=True)
        ids = torch.zeros(3, dtype=I32, device=cuda_device)
        with torch.no_grad():
            r = mtp_b200.route_tokens(x, 2)
            assert not any(t.requires_grad for t in (*r, mtp_b200.layer_norm(x), mtp_b200.embed_tokens(ids, x)))
        r = mtp_b200.route_tokens(x, 2)
        assert [t.requires_grad for t in r] == [True, False, False, True, True]

    def test_changed_inputs_are_noticed(self, cuda_device):
        """Saved tensors that a caller writes over before the backward pass."""
        x = torch.randn(6, 8, device=cuda_device, requires_grad=True)
        r = mtp_b200.route_tokens(x, 2)
        r.ids.add_(1)
        with pytest.raises(RuntimeError, match="modified"):
            r.weights.sum().backward()
        r = mtp_b200.route_tokens(x, 2)
        r.counts.zero_()  # as a reduction over ranks does: the gradient has its own
        r.balance_loss.backward()
        ids = torch.zeros(3, dtype=I32, device=cuda_device)
        out = mtp_b200.embed_tokens(ids, x)
        ids.add_(1)
        with pytest.raises(RuntimeError, match="modified"):
            out.sum().backward()

    @pytest.mark.parametrize("value", [1e39, -1e39, 10 ** 400])
    def test_numbers_that_fp32_does_not_hold(self, cuda_device, value):
        x, ids = torch.zeros(4, 8, device=cuda_device), torch.zeros(3, dtype=I32, device=cuda_device)
        with pytest.raises(ValueError, match="fp32"):
            mtp_b200.embed_tokens(ids, x, value)
        with pytest.raises(ValueError, match="fp32"):
            mtp_b200.layer_norm(x, eps=abs(value))

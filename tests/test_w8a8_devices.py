"""Token sort and int8 calls on tensors of a GPU that is not the current one: the device is current at the launch,
the stream is that device's, and the caller's device is current again afterwards. On the CPU, with fake tensors and
recorded entries."""
import contextlib

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mtp_b200
from mtp_b200 import w8a8

I32, I8 = torch.int32, torch.int8


class Entries:
    """Stands for the C entries: what was called, and which device was current then."""

    def __init__(self, monkeypatch, current):
        self.current, self.calls = current, []
        for name in ("sort", "unsort", "unsort_backward", "quantize", "matmul", "layer"):
            monkeypatch.setattr(w8a8, f"_{name}_entry", lambda *args, name=name: self.calls.append((name, self.current, args[-1])))
        monkeypatch.setattr(w8a8, "_current_device", lambda: self.current, raising=False)
        monkeypatch.setattr(w8a8, "_stream", lambda device: 1000 + device)
        monkeypatch.setattr(torch.cuda, "device", self.device)
        # fake tensors of a GPU that is not there, wherever this runs
        monkeypatch.setattr(torch.cuda, "is_available", lambda: False)

    @contextlib.contextmanager
    def device(self, index):
        before, self.current = self.current, index
        try:
            yield
        finally:
            self.current = before


def calls(z):
    """(entry, call) of every public function, on tensors that z makes."""
    x, ids, w = z(4, 16), z(4, 2, dtype=I32), z(4, 2)
    a, sa, b, sb = z(4, 16, dtype=I8), z(4), z(6, 16, dtype=I8), z(6)
    w13, s13, w2, s2 = z(3, 8, 16, dtype=I8), z(3, 8), z(3, 16, 4, dtype=I8), z(3, 16)
    return [
        ("sort", lambda: mtp_b200.sort_tokens(x, ids, 3)),
        ("unsort", lambda: mtp_b200.unsort_tokens(z(8, 16), ids, w)),
        ("unsort_backward", lambda: w8a8._unsort_backward(x, z(8, 16), 8, ids, w, True, True)),
        ("quantize", lambda: mtp_b200.quantize_int8(x)),
        ("matmul", lambda: mtp_b200.int8_matmul(a, sa, b, sb)),
        ("matmul", lambda: mtp_b200.int8_linear(x, b, sb)),
        ("matmul", lambda: mtp_b200.int8_grouped_matmul(a, sa, z(2, 6, 16, dtype=I8), z(2, 6), z(3, dtype=I32))),
        ("layer", lambda: mtp_b200.moe_layer_w8a8(x, z(4, 3), w13, s13, w2, s2, 2)),
        ("layer", lambda: mtp_b200.moe_layer_w8a8(x, None, w13, s13, w2, s2, 2, topk_weights=w, topk_ids=ids)),
    ]


@pytest.mark.filterwarnings("ignore:Accessing the data pointer of FakeTensor")
@pytest.mark.parametrize("index,current", [(1, 0), (0, 0), (0, 3)])
def test_the_tensors_device_is_current_at_the_launch(built_lib, monkeypatch, index, current):
    entries = Entries(monkeypatch, current)
    with FakeTensorMode():
        z = lambda *shape, dtype=torch.float32: torch.empty(*shape, dtype=dtype, device=f"cuda:{index}")
        for name, call in calls(z):
            entries.calls.clear()
            call()
            assert entries.calls == [(name, index, 1000 + index)]
            assert entries.current == current


@pytest.mark.gpu
def test_results_under_another_current_device(cuda_device, monkeypatch):
    """As if the current device were another: the tensors' own is entered, and the results are the same."""
    g = torch.Generator(device=cuda_device).manual_seed(0)
    x = torch.randn(40, 64, generator=g, device=cuda_device)
    ids = torch.randint(0, 5, (40, 2), generator=g, device=cuda_device, dtype=I32)

    def results():
        r = mtp_b200.sort_tokens(x, ids, 5)
        q, s = mtp_b200.quantize_int8(r.rows)
        b = torch.arange(5 * 32 * 64, device=cuda_device).remainder(127).to(I8).view(5, 32, 64)
        y = mtp_b200.int8_grouped_matmul(q, s, b, torch.ones(5, 32, device=cuda_device), r.offsets, out_dtype=torch.float32)
        return mtp_b200.unsort_tokens(y, r.positions)

    want = results()
    entered, current, device = [], [5], torch.cuda.device

    @contextlib.contextmanager
    def enter(index):
        entered.append(index)
        current.append(index)
        with device(index):
            yield
        current.pop()

    monkeypatch.setattr(w8a8, "_current_device", lambda: current[-1])
    monkeypatch.setattr(torch.cuda, "device", enter)
    got = results()
    assert entered == [0] * 4
    assert torch.equal(got, want)

"""Sizes that the kernels' 32-bit indexes do not hold are refused before a launch: at the C entries from
2^31 - 65535 on (their loops step past the last element by up to 32768), and in Python, whose ctypes would cut
2^32 + 8 to 8 without a word."""
import ctypes as C

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

LIMIT = 2 ** 31 - 65536
SHAPE, LAST = 2, 2 ** 31 - 1


@pytest.fixture
def entries(built_lib):
    """The C entries as functions of the sizes alone; one pointer for every buffer, which no refused call reads."""
    from mtp_b200 import _lib
    lib = _lib.load()
    buf = (C.c_uint8 * 1024)()
    p = C.addressof(buf) + (-C.addressof(buf)) % 256

    def sort(m=2, h=8, k=2):
        return lib.mtp_sort_tokens(p, h, 0, m, h, p, k, 4, None, 0, None, p, None, p, p, None)

    def unsort(m=2, h=8, k=2, rows=None):
        return lib.mtp_unsort_tokens(p, m * k if rows is None else rows, 0, p, None, m, k, h, p, None)

    def backward(m=2, h=8, k=2, rows=None):
        return lib.mtp_unsort_tokens_backward(p, p, m * k if rows is None else rows, 0, p, None, m, k, h, p, None, None)

    def quantize(m=2, k=8):
        return lib.mtp_quantize_int8(p, k, 0, m, k, p, k, p, None)

    def matmul(m=2, n=8, groups=1):
        args = _lib.MtpInt8MatmulArgs(rows=m, n=n, k=16, num_groups=groups, a_dtype=3, out_dtype=0, a=p, a_stride=16,
                                      a_scale=p, b=p, b_scale=p, offsets=p if groups > 1 else None, out=p)
        return lib.mtp_int8_matmul(C.byref(args), None)

    def matmul_size(m=2, n=8, groups=1):
        args = _lib.MtpInt8MatmulArgs(rows=m, n=n, k=16, num_groups=groups, a_dtype=3, a=p, a_stride=16, b=p,
                                      offsets=p if groups > 1 else None)
        return lib.mtp_int8_matmul_workspace_size(C.byref(args), C.byref(C.c_int64()))

    def layer_size(m=2, h=16, i=16, e=4, k=2):
        args = _lib.MtpW8A8LayerArgs(num_tokens=m, hidden=h, inter=i, num_experts=e, top_k=k, dtype=0, hidden_states=p,
                                     w13=p, w2=p)
        return lib.mtp_w8a8_moe_layer_workspace_size(C.byref(args), C.byref(C.c_int64()))

    return locals()


@pytest.mark.parametrize("name,sizes", [
    ("sort", dict(h=LAST)), ("sort", dict(h=LIMIT + 1)), ("sort", dict(m=LAST - 1, k=1)), ("sort", dict(m=2 ** 26, k=32)),
    ("sort", dict(m=LIMIT + 1, k=1)),
    ("unsort", dict(h=LAST)), ("unsort", dict(h=LIMIT + 1)), ("unsort", dict(m=LIMIT + 1, k=1)), ("unsort", dict(rows=LIMIT + 1)),
    ("backward", dict(h=LAST)), ("backward", dict(h=LIMIT + 1)), ("backward", dict(m=LIMIT + 1, k=1)),
    ("backward", dict(rows=LIMIT + 1)),
    ("quantize", dict(k=LAST)), ("quantize", dict(k=LIMIT + 1)), ("quantize", dict(m=LAST)), ("quantize", dict(m=LIMIT + 1)),
    ("matmul", dict(m=LAST)), ("matmul", dict(m=LIMIT + 1)), ("matmul", dict(n=LAST)), ("matmul", dict(n=LIMIT + 1)),
    ("matmul", dict(n=2 ** 21, groups=1024)), ("matmul_size", dict(m=LIMIT + 1)), ("matmul_size", dict(n=LIMIT + 1)),
    ("layer_size", dict(m=LIMIT + 1, k=1)), ("layer_size", dict(m=2 ** 26, k=32)),
])
def test_c_entries_refuse_what_32_bits_do_not_index(entries, name, sizes):
    assert entries[name](**sizes) == SHAPE


def test_c_entries_take_the_largest_sizes(entries):
    """The workspace queries, which launch nothing, at the limit itself."""
    assert entries["matmul_size"](m=LIMIT) == 0
    assert entries["matmul_size"](n=LIMIT) == 0
    assert entries["matmul_size"](n=2 ** 21 - 64, groups=1024) == 0
    assert entries["layer_size"](m=LIMIT, k=1) == 0
    assert entries["layer_size"](m=LIMIT // 8, k=8) == 0


I32, I8, BF = torch.int32, torch.int8, torch.bfloat16


def calls(z, n):
    """Every public function with a size of n, on tensors that z makes."""
    import mtp_b200 as p
    ids = z(2, 1, dtype=I32)
    layer = (z(3, 8, 16, dtype=I8), z(3, 8), z(3, 16, 4, dtype=I8), z(3, 16), 1)
    return {
        "sort columns": lambda: p.sort_tokens(z(2, n, dtype=BF), ids, 3),
        "sort pairs": lambda: p.sort_tokens(z(n, 4, dtype=BF), z(n, 1, dtype=I32), 3),
        "sort map": lambda: p.sort_tokens(z(2, 4), ids, 3, expert_map=z(n, dtype=I32)),
        "unsort columns": lambda: p.unsort_tokens(z(2, n, dtype=BF), ids),
        "unsort pairs": lambda: p.unsort_tokens(z(n, 4, dtype=BF), z(n, 1, dtype=I32)),
        "quantize columns": lambda: p.quantize_int8(z(1, n, dtype=BF)),
        "quantize rows": lambda: p.quantize_int8(z(n, 1, dtype=BF)),
        "matmul rows": lambda: p.int8_matmul(z(n, 16, dtype=I8), z(n), z(4, 16, dtype=I8), z(4)),
        "matmul channels": lambda: p.int8_matmul(z(2, 16, dtype=I8), z(2), z(n, 16, dtype=I8), z(n)),
        "linear rows": lambda: p.int8_linear(z(n, 16), z(4, 16, dtype=I8), z(4)),
        "grouped rows": lambda: p.int8_grouped_matmul(z(n, 16, dtype=I8), z(n), z(1, 4, 16, dtype=I8), z(1, 4), z(2, dtype=I32)),
        "grouped channels": lambda: p.int8_grouped_matmul(z(2, 16, dtype=I8), z(2), z(4, n, 16, dtype=I8), z(4, n), z(5, dtype=I32)),
        "layer tokens": lambda: p.moe_layer_w8a8(z(n, 16), z(n, 3), *layer),
        "layer map": lambda: p.moe_layer_w8a8(z(2, 16), None, *layer, topk_weights=z(2, 1), topk_ids=ids, expert_map=z(n, dtype=I32)),
    }


@pytest.mark.filterwarnings("ignore:Accessing the data pointer of FakeTensor")
@pytest.mark.parametrize("n", [LIMIT + 1, 2 ** 31, 2 ** 32 + 8])
def test_python_refuses_what_32_bits_do_not_index(built_lib, monkeypatch, n):
    from mtp_b200 import w8a8
    for entry in ("sort", "unsort", "quantize", "matmul", "layer"):
        monkeypatch.setattr(w8a8, f"_{entry}_entry", lambda *args: None)
    monkeypatch.setattr(w8a8, "_current_device", lambda: 0, raising=False)
    monkeypatch.setattr(w8a8, "_stream", lambda device: 0)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: False)
    taken = []
    with FakeTensorMode():
        z = lambda *shape, dtype=torch.float32: torch.empty(*shape, dtype=dtype, device="cuda:0")
        for name, call in calls(z, n).items():
            try:
                call()
                taken.append(name)
            except ValueError as e:
                assert "supported" in str(e), name
    assert not taken

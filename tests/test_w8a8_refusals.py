"""What the token sort and the int8 products refuse, in Python before a launch
and at the C entries with a status. CPU only."""
import ctypes as C

import pytest
import torch


def call(name, *args, **kw):
    import mtp_b200
    return getattr(mtp_b200, name)(*args, **kw)


I32, I8, BF = torch.int32, torch.int8, torch.bfloat16


@pytest.mark.parametrize("name,args", [
    ("sort_tokens", (torch.zeros(2, 4), torch.zeros(2, 1, dtype=I32), 4)),
    ("unsort_tokens", (torch.zeros(2, 4), torch.zeros(2, 1, dtype=I32))),
    ("quantize_int8", (torch.zeros(2, 4),)),
    ("int8_matmul", (torch.zeros(2, 16, dtype=I8), torch.zeros(2), torch.zeros(4, 16, dtype=I8), torch.zeros(4))),
    ("int8_linear", (torch.zeros(2, 16), torch.zeros(4, 16, dtype=I8), torch.zeros(4))),
    ("int8_grouped_matmul", (torch.zeros(2, 16, dtype=I8), torch.zeros(2), torch.zeros(1, 4, 16, dtype=I8),
                             torch.zeros(1, 4), torch.zeros(2, dtype=I32))),
    ("moe_layer_w8a8", (torch.zeros(2, 16), torch.zeros(2, 4), torch.zeros(4, 8, 16, dtype=I8), torch.zeros(4, 8),
                        torch.zeros(4, 16, 4, dtype=I8), torch.zeros(4, 16), 2)),
])
def test_host_tensors_are_refused(built_lib, name, args):
    with pytest.raises(ValueError, match="CUDA"):
        call(name, *args)
    with pytest.raises(TypeError):
        call(name, [1.0], *args[1:])


def test_c_entries_answer_bad_arguments_without_a_gpu(built_lib):
    from mtp_b200 import _lib
    lib = _lib.load()
    buf = (C.c_uint8 * 4096)()
    p = C.addressof(buf) + (-C.addressof(buf)) % 256
    sort = lambda x=p, stride=8, dt=0, m=2, h=8, ids=p, k=2, e=4, emap=None, ge=0, rs=None, rows=p, ss=None, pos=p, off=p: (
        lib.mtp_sort_tokens(x, stride, dt, m, h, ids, k, e, emap, ge, rs, rows, ss, pos, off, None))
    assert sort(ids=None) == 1 and sort(pos=None) == 1 and sort(off=None) == 1 and sort(rows=None) == 1
    assert sort(rs=p) == 1                                      # scales without room for the sorted ones
    for bad in (dict(m=-1), dict(k=0), dict(k=33), dict(e=0), dict(e=1025), dict(h=-1), dict(m=2 ** 27, k=32),
                dict(emap=p, ge=0), dict(stride=-1)):
        assert sort(**bad) == 2, bad
    assert sort(dt=4) == 9 and sort(x=p + 1) == 3 and sort(rows=p + 1) == 3

    unsort = lambda rows=p, n=4, dt=0, pos=p, w=None, m=2, k=2, h=8, out=p: (
        lib.mtp_unsort_tokens(rows, n, dt, pos, w, m, k, h, out, None))
    assert unsort(rows=None) == 1 and unsort(pos=None) == 1 and unsort(out=None) == 1
    assert unsort(k=33) == 2 and unsort(n=-1) == 2 and unsort(n=2 ** 31) == 2 and unsort(m=-1) == 2
    assert unsort(dt=3) == 9 and unsort(out=p + 1) == 3
    assert unsort(m=0) == 0

    back = lambda g=p, rows=p, n=4, dt=0, pos=p, w=None, m=2, k=2, h=8, gr=p, gw=p: (
        lib.mtp_unsort_tokens_backward(g, rows, n, dt, pos, w, m, k, h, gr, gw, None))
    assert back(g=None) == 1 and back(rows=None) == 1 and back(pos=None) == 1
    assert back(k=0) == 2 and back(dt=3) == 9 and back(gr=p + 1) == 3
    assert back(gr=None, gw=None) == 0

    quant = lambda x=p, stride=8, dt=0, m=2, k=8, q=p, qs=8, s=p: lib.mtp_quantize_int8(x, stride, dt, m, k, q, qs, s, None)
    assert quant(x=None) == 1 and quant(q=None) == 1 and quant(s=None) == 1
    assert quant(k=0) == 2 and quant(qs=7) == 2 and quant(m=-1) == 2 and quant(dt=3) == 9 and quant(x=p + 1) == 3
    assert quant(m=0) == 0

    base = dict(rows=2, n=8, k=16, num_groups=1, a_dtype=3, out_dtype=0, a=p, a_stride=16, a_scale=p, b=p, b_scale=p, out=p)

    def matmul(**kw):
        args = _lib.MtpInt8MatmulArgs(**{**base, **kw})
        return lib.mtp_int8_matmul(C.byref(args), None)
    assert lib.mtp_int8_matmul(None, None) == 1
    for name in ("a", "a_scale", "b", "b_scale", "out"):
        assert matmul(**{name: None}) == 1, name
    for bad in (dict(rows=-1), dict(n=0), dict(k=0), dict(k=131072, a_stride=131072), dict(num_groups=0), dict(num_groups=2),
                dict(num_groups=1025, offsets=p), dict(a_stride=15), dict(activation=1, n=7), dict(activation=1, bias=p),
                dict(n=2 ** 30, num_groups=2, offsets=p)):
        assert matmul(**bad) == 2, bad
    assert matmul(a_dtype=4) == 9 and matmul(out_dtype=3) == 9 and matmul(activation=2) == 9
    assert matmul(out=p + 1) == 3 and matmul(workspace=p + 16, workspace_bytes=4096) == 3
    assert matmul(rows=20, a_dtype=0, a_scale=None) == 1         # more than a few rows are quantised in a workspace
    assert matmul(rows=20, a_dtype=0, a_scale=None, workspace=p, workspace_bytes=16) == 4
    assert matmul(rows=0, a=None, b=None, out=None) == 0

    need = C.c_int64()
    args = _lib.MtpInt8MatmulArgs(**base)
    assert lib.mtp_int8_matmul_workspace_size(C.byref(args), C.byref(need)) == 0 and need.value == 0
    args.a = p + 8                                              # not a row start that TMA takes
    assert lib.mtp_int8_matmul_workspace_size(C.byref(args), C.byref(need)) == 0 and need.value >= 2 * 16
    assert lib.mtp_int8_matmul_workspace_size(C.byref(args), None) == 1

    layer = dict(num_tokens=2, hidden=16, inter=16, num_experts=4, top_k=2, dtype=0, hidden_states=p, router_logits=p,
                 w13=p, w13_scale=p, w2=p, w2_scale=p, out=p, workspace=p, workspace_bytes=1 << 40)

    def moe(**kw):
        args = _lib.MtpW8A8LayerArgs(**{**layer, **kw})
        return lib.mtp_w8a8_moe_layer(C.byref(args), None)
    assert lib.mtp_w8a8_moe_layer(None, None) == 1
    for name in ("hidden_states", "router_logits", "w13", "w13_scale", "w2", "w2_scale", "out", "workspace"):
        assert moe(**{name: None}) == 1, name
    for bad in (dict(num_tokens=-1), dict(hidden=0), dict(inter=0), dict(num_experts=0), dict(num_experts=1025),
                dict(top_k=0), dict(top_k=5), dict(top_k=33), dict(hidden=131072),
                dict(router_logits=None, expert_map=p, global_num_experts=0)):
        assert moe(**bad) == 2, bad
    assert moe(expert_map=p, global_num_experts=4) == 9          # a map needs given ids
    assert moe(dtype=3) == 9 and moe(workspace_bytes=64) == 4 and moe(out=p + 1) == 3
    assert moe(num_tokens=0) == 0


class TestOnTheGpu:
    pytestmark = pytest.mark.gpu

    def test_shapes_types_and_layouts(self, cuda_device):
        z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device=cuda_device)
        x, ids = z(4, 8), z(4, 2, dtype=I32)
        bad = [
            ("sort_tokens", (x, ids[:3], 4), {}), ("sort_tokens", (x, ids.long(), 4), {}), ("sort_tokens", (x, ids, 0), {}),
            ("sort_tokens", (x, ids, 1025), {}), ("sort_tokens", (x.double(), ids, 4), {}),
            ("sort_tokens", (x, z(4, 33, dtype=I32), 4), {}), ("sort_tokens", (x, z(4, 0, dtype=I32), 4), {}),
            ("sort_tokens", (x.t(), z(8, 2, dtype=I32), 4), {}), ("sort_tokens", (x[:1].expand(4, 8), ids, 4), {}),
            ("sort_tokens", (x, ids, 4), dict(row_scales=z(3))), ("sort_tokens", (x, ids, 4), dict(expert_map=z(0, dtype=I32))),
            ("sort_tokens", (x, ids, 4), dict(expert_map=z(4))),
            ("unsort_tokens", (z(7, 8), ids), {}), ("unsort_tokens", (z(8, 8, dtype=I8), ids), {}),
            ("unsort_tokens", (z(8, 8), ids.long()), {}), ("unsort_tokens", (z(8, 8), ids, z(4, 3)), {}),
            ("unsort_tokens", (z(8, 8), ids, z(4, 2, dtype=BF)), {}), ("unsort_tokens", (z(8, 16)[:, :8], ids), {}),
            ("quantize_int8", (z(4, 0),), {}), ("quantize_int8", (z(4, 8).t(),), {}), ("quantize_int8", (z(4, 8, dtype=I8),), {}),
        ]
        a, sa, b, sb = z(4, 16, dtype=I8), z(4), z(6, 16, dtype=I8), z(6)
        bad += [
            ("int8_matmul", (a, sa, b[:, :8].contiguous(), sb), {}), ("int8_matmul", (a, sa[:3], b, sb), {}),
            ("int8_matmul", (a, sa, b, sb[:5]), {}), ("int8_matmul", (a, sa, b.t(), sb), {}),
            ("int8_matmul", (a.float(), sa, b, sb), {}), ("int8_matmul", (a, sa, b, sb), dict(bias=z(5))),
            ("int8_matmul", (a, sa, b, sb), dict(bias=z(6, dtype=BF))), ("int8_matmul", (a, sa, b, sb), dict(out_dtype=I8)),
            ("int8_matmul", (a, sa, b, sb.to(BF)), {}), ("int8_matmul", (a, sa, b[:0], sb[:0]), {}),
            ("int8_matmul", (a, sa, b, sb), dict(status=z(0, dtype=I32))), ("int8_matmul", (a.t(), z(16), z(6, 4, dtype=I8), sb), {}),
            ("int8_matmul", (z(2, 131072, dtype=I8), z(2), z(1, 131072, dtype=I8), z(1)), {}),
            ("int8_linear", (a, b, sb), {}), ("int8_linear", (z(4, 15), b, sb), {}),
            ("int8_grouped_matmul", (a, sa, b[None], sb[None], z(3, dtype=I32)), {}),
            ("int8_grouped_matmul", (a, sa, b, sb, z(2, dtype=I32)), {}),
            ("int8_grouped_matmul", (a, sa, b[None], sb[None], z(2)), {}),
            ("int8_grouped_matmul", (a, sa, b[None, :5].contiguous(), sb[None, :5].contiguous(), z(2, dtype=I32)), dict(activation="silu_mul")),
            ("int8_grouped_matmul", (a, sa, b[None], sb[None], z(2, dtype=I32)), dict(activation="gelu")),
            ("int8_grouped_matmul", (a, sa, z(1025, 2, 16, dtype=I8), z(1025, 2), z(1026, dtype=I32)), {}),
        ]
        x, lg = z(4, 16), z(4, 3)
        w13, s13, w2, s2 = z(3, 8, 16, dtype=I8), z(3, 8), z(3, 16, 4, dtype=I8), z(3, 16)
        w, i = z(4, 2), z(4, 2, dtype=I32)
        bad += [("moe_layer_w8a8", args, kw) for args, kw in [
            ((x, lg, w13, s13, w2, s2, 4), {}), ((x, lg, w13, s13, w2, s2, 0), {}), ((x, lg[:, :2].contiguous(), w13, s13, w2, s2, 2), {}),
            ((x, lg, w13[:, :7].contiguous(), s13[:, :7].contiguous(), w2, s2, 2), {}), ((x, lg, w13, s13, w2[:2], s2[:2], 2), {}),
            ((x, lg, w13, s13[:2], w2, s2, 2), {}), ((x.t(), lg, w13, s13, w2, s2, 2), {}),
            ((x, None, w13, s13, w2, s2, 2), {}), ((x, None, w13, s13, w2, s2, 2), dict(topk_weights=w, topk_ids=i.long())),
            ((x, None, w13, s13, w2, s2, 1), dict(topk_weights=w, topk_ids=i)),
            ((x, lg, w13, s13, w2, s2, 2), dict(expert_map=z(3, dtype=I32))),
            ((x, lg, w13, s13, w2, s2, 2), dict(out=z(4, 16, dtype=BF))), ((x, lg, w13, s13, w2, s2, 2), dict(out=z(3, 16)))]]
        for name, args, kw in bad:
            with pytest.raises(ValueError):
                call(name, *args, **kw)
                pytest.fail(f"{name} took {[tuple(getattr(t, 'shape', [t])) for t in args]} {sorted(kw)}")

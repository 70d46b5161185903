"""The int8 (W8A8) expert path and the token sort around it: torch tensors in,
C-ABI calls out.

* :func:`sort_tokens` / :func:`unsort_tokens` - token rows into expert order and
  back with the routing weights applied; both have gradients
  (``torch.autograd``);
* :func:`quantize_int8` - rows to int8 codes with one scale each;
* :func:`int8_matmul` / :func:`int8_linear` - int8 rows (or rows quantised on the
  way in) times int8 weights with one scale per output channel;
* :func:`int8_grouped_matmul` - the same with one weight matrix per group of
  sorted rows, optionally with SiLU(gate) * up;
* :func:`moe_layer_w8a8` - router, sort, both expert products and the way back.

Pair order, ``-1`` ids and ``expert_map`` follow :func:`mtp_b200.moe_align_block_size`
and :func:`mtp_b200.moe_layer_w4a16`. Shape, dtype and device errors raise
``ValueError`` before any launch; a non-zero C status raises
:class:`mtp_b200.MtpError`. Every call is asynchronous on the current torch
stream of its tensors' GPU, which need not be the current one. There is no CPU
path. Only the token sort has gradients: the other functions work on inputs that
require one, but a backward pass that reaches them raises ``NotImplementedError``.
"""
from __future__ import annotations

import ctypes as C
from functools import lru_cache
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _lib

DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}  # MtpDtype
_INT8 = 3
MAX_K = 131071  # 128 * 128 * K stays below 2^31
MAX_EXTENT = 2 ** 31 - 65536  # rows, columns, pairs and channels of a call (ctypes would cut larger ones to 32 bits)
_SILU_MUL = 1


_sort_entry = _lib.Entry("mtp_sort_tokens")
_unsort_entry = _lib.Entry("mtp_unsort_tokens")
_unsort_backward_entry = _lib.Entry("mtp_unsort_tokens_backward")
_quantize_entry = _lib.Entry("mtp_quantize_int8")
_matmul_entry = _lib.Entry("mtp_int8_matmul")
_layer_entry = _lib.Entry("mtp_w8a8_moe_layer")

# The current device, on which the C side launches: the functions below that launch make their tensors' device
# current first. And the handle of a device's current stream (torch.cuda.current_stream builds a Stream object around it).
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_stream = (getattr(torch._C, "_cuda_getCurrentRawStream", None)
           or (lambda device: torch.cuda.current_stream(device).cuda_stream))


def _tensor(name: str, t, ndim: int, dtypes, device: torch.device | None = None, contiguous: bool = True):
    """``t`` is a CUDA tensor of one of ``dtypes`` and ``ndim`` dimensions on ``device``."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if device is None or t.device != device:
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor, got device {t.device}")
        if device is not None:
            raise ValueError(f"{name} is on {t.device}, expected {device}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be one of {[str(d) for d in dtypes]}, got {t.dtype}")
    if t.ndim != ndim:
        raise ValueError(f"{name} must be {ndim}-D, got shape {tuple(t.shape)}")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _too_large(what: str, n: int):
    raise ValueError(f"at most {MAX_EXTENT} {what} are supported, got {n}")


def _check_map(expert_map: torch.Tensor, device: torch.device):
    _tensor("expert_map", expert_map, 1, _I32, device)
    if not expert_map.numel():
        raise ValueError("expert_map is empty")
    if expert_map.numel() > MAX_EXTENT:
        _too_large("entries of expert_map", expert_map.numel())


def _differentiated(*tensors) -> bool:
    """Whether a derivative of one of ``tensors`` is being recorded, backward or (dual tensors) forward."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    if forward_ad._current_level < 0:  # outside dual_level there are no duals (unpack_dual takes 0.3 us)
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


class _NoGradient(torch.autograd.Function):
    """call(), whose derivatives with respect to ``inputs`` are errors instead of missing."""

    @staticmethod
    def forward(ctx, name, call, *inputs):
        ctx.name = name
        return call()

    @staticmethod
    def backward(ctx, *grads):
        raise NotImplementedError(f"{ctx.name} has no gradient")


_F32 = (torch.float32,)
_I32 = (torch.int32,)
_I8 = (torch.int8,)
_ROWS = (torch.bfloat16, torch.float16, torch.float32, torch.int8)
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


def _row_stride(name: str, t: torch.Tensor) -> int:
    """Elements between the rows of a 2-D tensor whose rows are contiguous and do not overlap."""
    if t.is_contiguous():
        return t.shape[1]
    if t.shape[0] <= 1:
        if t.shape[1] > 1 and t.stride(1) != 1:
            raise ValueError(f"the rows of {name} must be contiguous")
        return t.shape[1]
    if (t.shape[1] > 1 and t.stride(1) != 1) or t.stride(0) < t.shape[1]:
        raise ValueError(f"the rows of {name} must be contiguous and must not overlap, got strides {t.stride()}")
    return t.stride(0)


# ---------------------------------------------------------------------------
# sort and unsort
# ---------------------------------------------------------------------------
class SortedTokens(NamedTuple):
    """What :func:`sort_tokens` returns.

    ``rows`` [M*k, H] in expert order (pairs without an expert last, as zeros),
    ``positions`` [M, k] int32 (the pair's row, or ``~row`` < 0 without an
    expert), ``offsets`` [E + 1] int32 (first row of each expert, then the
    number of routed rows), ``row_scales`` [M*k] fp32 if scales were given."""

    rows: torch.Tensor
    positions: torch.Tensor
    offsets: torch.Tensor
    row_scales: torch.Tensor | None


def _sort(x, ids, num_experts, expert_map, row_scales):
    device = x.get_device()
    if device != _current_device():
        with torch.cuda.device(device):
            return _sort(x, ids, num_experts, expert_map, row_scales)
    m, k = ids.shape
    h = x.shape[1]
    rows = x.new_empty(m * k, h)
    positions = torch.empty_like(ids)
    offsets = ids.new_empty(num_experts + 1)
    scales = None if row_scales is None else row_scales.new_empty(m * k)
    _sort_entry(x.data_ptr() or None, _row_stride("hidden_states", x), DTYPES.get(x.dtype, _INT8), m, h,
              ids.data_ptr(), k, num_experts, None if expert_map is None else expert_map.data_ptr(),
              0 if expert_map is None else expert_map.numel(), None if scales is None else row_scales.data_ptr(),
              rows.data_ptr(), None if scales is None else scales.data_ptr(), positions.data_ptr(),
              offsets.data_ptr(), _stream(device))
    return rows, positions, offsets, scales


def _unsort(rows, positions, weights):
    device = rows.get_device()
    if device != _current_device():
        with torch.cuda.device(device):
            return _unsort(rows, positions, weights)
    m, k = positions.shape
    r, h = rows.shape
    out = rows.new_empty(m, h)
    _unsort_entry(rows.data_ptr(), r, DTYPES[rows.dtype], positions.data_ptr(),
                  None if weights is None else weights.data_ptr(), m, k, h, out.data_ptr(), _stream(device))
    return out


def _unsort_backward(grad, rows, num_rows, positions, weights, need_rows, need_weights):
    device = grad.get_device()
    if device != _current_device():
        with torch.cuda.device(device):
            return _unsort_backward(grad, rows, num_rows, positions, weights, need_rows, need_weights)
    (m, k), h = positions.shape, grad.shape[1]
    grad_rows = grad.new_empty(num_rows, h) if need_rows else None
    grad_weights = torch.empty_like(weights) if need_weights else None
    _unsort_backward_entry(grad.data_ptr(), None if rows is None else rows.data_ptr(), num_rows, DTYPES[grad.dtype],
                           positions.data_ptr(), None if weights is None else weights.data_ptr(), m, k, h,
                           None if grad_rows is None else grad_rows.data_ptr(),
                           None if grad_weights is None else grad_weights.data_ptr(), _stream(device))
    return grad_rows, grad_weights


class _SortTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, ids, num_experts, expert_map, row_scales, rest):
        # positions, offsets and scales are not differentiable: they go around autograd, in `rest`
        rows, *others = _sort(x, ids, num_experts, expert_map, row_scales)
        ctx.save_for_backward(others[0])
        rest.extend(others)
        return rows

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_rows):
        (positions,) = ctx.saved_tensors
        return _unsort(grad_rows.contiguous(), positions, None), None, None, None, None, None


class _UnsortTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, positions, weights):
        ctx.save_for_backward(rows if weights is not None and weights.requires_grad else None, positions, weights)
        ctx.num_rows = rows.shape[0]
        return _unsort(rows, positions, weights)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        rows, positions, weights = ctx.saved_tensors
        need_rows, _, need_weights = ctx.needs_input_grad
        grad_rows, grad_weights = _unsort_backward(grad.contiguous(), rows, ctx.num_rows, positions, weights, need_rows,
                                                   need_weights)
        return grad_rows, None, grad_weights


def sort_tokens(hidden_states: torch.Tensor, topk_ids: torch.Tensor, num_experts: int, *,
                expert_map: torch.Tensor | None = None, row_scales: torch.Tensor | None = None) -> SortedTokens:
    """The rows of ``hidden_states`` [M, H] (bf16, fp16, fp32 or int8) in expert
    order, one per pair of a token and one of its ``topk_ids`` [M, k] int32.

    The order is stable (experts ascending, ``t*k + j`` ascending inside an
    expert). Ids outside [0, ``num_experts``) - after ``expert_map`` [global E]
    int32, if given - have no expert here: their rows come last, as zeros.
    ``row_scales`` [M] fp32 (the scales of int8 rows) are sorted along. The
    gradient of ``hidden_states`` sums the gradients of a token's routed rows
    in fp32. Forward-mode derivatives raise ``RuntimeError``."""
    _tensor("hidden_states", hidden_states, 2, _ROWS, contiguous=False)
    dev = hidden_states.device
    _tensor("topk_ids", topk_ids, 2, _I32, dev)
    (m, k), (tokens, h) = topk_ids.shape, hidden_states.shape
    if m != tokens:
        raise ValueError(f"topk_ids has {m} rows, hidden_states has {tokens}")
    if not 1 <= k <= 32:
        raise ValueError(f"topk_ids must have 1 to 32 columns, got {k}")
    if not 1 <= num_experts <= 1024:
        raise ValueError(f"num_experts must be in [1, 1024], got {num_experts}")
    if m * k > MAX_EXTENT:
        _too_large("pairs", m * k)
    if h > MAX_EXTENT:
        _too_large("columns", h)
    if expert_map is not None:
        _check_map(expert_map, dev)
    if row_scales is not None:
        _tensor("row_scales", row_scales, 1, _F32, dev)
        if row_scales.numel() != m:
            raise ValueError(f"row_scales must have {m} entries")
    if _differentiated(hidden_states):
        rest = []
        r = SortedTokens(_SortTokens.apply(hidden_states, topk_ids, num_experts, expert_map, row_scales, rest), *rest)
    else:
        r = SortedTokens(*_sort(hidden_states, topk_ids, num_experts, expert_map, row_scales))
    if row_scales is not None and _differentiated(row_scales):
        r = r._replace(row_scales=_NoGradient.apply("row_scales of sort_tokens", lambda: r.row_scales, row_scales))
    return r


def unsort_tokens(rows: torch.Tensor, positions: torch.Tensor,
                  topk_weights: torch.Tensor | None = None) -> torch.Tensor:
    """out [M, H] = the weighted sum of each token's routed ``rows`` [R, H] (bf16,
    fp16 or fp32), in fp32 and rounded once. ``positions`` [M, k] int32 as
    :func:`sort_tokens` gives them; ``topk_weights`` [M, k] fp32 (None: 1). A
    token without routed pairs gets zeros. Gradients go to ``rows`` (zero for
    rows of unrouted pairs) and ``topk_weights``; forward-mode derivatives raise
    ``RuntimeError``."""
    _tensor("rows", rows, 2, _FLOATS)
    _tensor("positions", positions, 2, _I32, rows.device)
    (m, k), (pairs, h) = positions.shape, rows.shape
    if not 1 <= k <= 32:
        raise ValueError(f"positions must have 1 to 32 columns, got {k}")
    if pairs != m * k:
        raise ValueError(f"rows must have one row per pair, {m * k}, got {pairs}")
    if pairs > MAX_EXTENT:
        _too_large("pairs", pairs)
    if h > MAX_EXTENT:
        _too_large("columns", h)
    if topk_weights is not None:
        _tensor("topk_weights", topk_weights, 2, _F32, rows.device)
        if topk_weights.shape != positions.shape:
            raise ValueError(f"topk_weights must be {(m, k)}, got {tuple(topk_weights.shape)}")
    if _differentiated(rows, topk_weights):
        return _UnsortTokens.apply(rows, positions, topk_weights)
    return _unsort(rows, positions, topk_weights)


# ---------------------------------------------------------------------------
# int8 products
# ---------------------------------------------------------------------------
def quantize_int8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(codes int8 [M, K], scales fp32 [M])`` of the rows of ``x`` [M, K] (bf16,
    fp16 or fp32): scale = max|x| / 127, code = round(x * (127 / max|x|)), half
    to even. A row of zeros has scale 0; a row with an infinity or a NaN has
    that as its scale and codes 0. The codes' rows are a multiple of 16 bytes
    apart, as the products read them best."""
    _tensor("x", x, 2, _FLOATS, contiguous=False)
    m, k = x.shape
    if k < 1:
        raise ValueError("x must have at least one column")
    if m > MAX_EXTENT:
        _too_large("rows", m)
    if k > MAX_EXTENT:
        _too_large("columns", k)
    if _differentiated(x):
        return _NoGradient.apply("quantize_int8", lambda: _quantize(x), x)
    return _quantize(x)


def _quantize(x):
    device = x.get_device()
    if device != _current_device():
        with torch.cuda.device(device):
            return _quantize(x)
    m, k = x.shape
    kp = (k + 15) // 16 * 16
    codes = x.new_empty(m, kp, dtype=torch.int8)
    scale = x.new_empty(m, dtype=torch.float32)
    _quantize_entry(x.data_ptr(), _row_stride("x", x), DTYPES[x.dtype], m, k, codes.data_ptr(), kp, scale.data_ptr(),
                    _stream(device))
    return codes if kp == k else codes[:, :k], scale


@lru_cache(maxsize=4096)
def _matmul_workspace(rows, n, k, groups, a_dtype, a_stride, a_off, b_off) -> int:
    """Workspace bytes; a_off and b_off are the operands' addresses modulo 256 (their alignment)."""
    args = _lib.MtpInt8MatmulArgs(rows, n, k, groups, a_dtype, 0, 0, 0, 256 + a_off, a_stride, None, 256 + b_off, None,
                                  None, 256 if groups > 1 else None, None, None, None, 0)
    out = _lib.i64()
    _lib.call("mtp_int8_matmul_workspace_size", C.byref(args), C.byref(out))
    return out.value


def _product(a, a_scale, b, b_scale, bias, offsets, shape, out_dtype, activation, status):
    device = a.get_device()
    if device != _current_device():
        with torch.cuda.device(device):
            return _product(a, a_scale, b, b_scale, bias, offsets, shape, out_dtype, activation, status)
    rows, k, groups, n = shape
    cols = n // 2 if activation else n
    out = a.new_empty(rows, cols) if out_dtype is a.dtype else a.new_empty(rows, cols, dtype=out_dtype)
    a_dtype, a_stride = DTYPES.get(a.dtype, _INT8), _row_stride("a", a)
    ap, bp = a.data_ptr(), b.data_ptr()
    size = _matmul_workspace(rows, n, k, groups, a_dtype, a_stride, ap & 255, bp & 255)
    ws = b.new_empty(size) if size else None
    args = _lib.MtpInt8MatmulArgs(rows, n, k, groups, a_dtype, DTYPES[out_dtype], activation, 0, ap, a_stride,
                                  None if a_scale is None else a_scale.data_ptr(), bp, b_scale.data_ptr(),
                                  None if bias is None else bias.data_ptr(),
                                  None if offsets is None else offsets.data_ptr(), out.data_ptr(),
                                  None if status is None else status.data_ptr(),
                                  None if ws is None else ws.data_ptr(), size)
    _matmul_entry(C.byref(args), _stream(device))
    return out


def _check_weight(name, b, scale, ndim, device, k):
    """Checks weights [(groups,) n, k] and their scales; returns (groups, n)."""
    _tensor(name, b, ndim, _I8, device)
    _tensor(name + "_scale", scale, ndim - 1, _F32, device)
    *lead, cols = b.shape
    if cols != k:
        raise ValueError(f"{name} must have {k} columns, got shape {tuple(b.shape)}")
    if list(scale.shape) != lead:
        raise ValueError(f"{name}_scale must be {tuple(lead)}, got {tuple(scale.shape)}")
    groups, n = lead if ndim == 3 else (1, lead[0])
    if not 1 <= k <= MAX_K:
        raise ValueError(f"1 to {MAX_K} columns are supported, got {k}")
    if not groups or not n:
        raise ValueError(f"{name} must not be empty, got shape {tuple(b.shape)}")
    if groups * n > MAX_EXTENT:
        _too_large(f"rows of {name}", groups * n)
    return groups, n


def _check_bias(bias, n, device):
    if bias is not None:
        _tensor("bias", bias, 1, _F32, device)
        if bias.numel() != n:
            raise ValueError(f"bias must have {n} entries")


def _check_out(out_dtype, status, device):
    if out_dtype not in DTYPES:
        raise ValueError(f"out_dtype must be one of {[str(d) for d in DTYPES]}, got {out_dtype}")
    if status is not None:
        _tensor("status", status, 1, _I32, device)
        if not status.numel():
            raise ValueError("status must have an entry")


def _check_rows(a, a_scale):
    """Checks int8 rows and their scales; returns (rows, k, device)."""
    _tensor("a", a, 2, _I8, contiguous=False)
    device = a.device
    _tensor("a_scale", a_scale, 1, _F32, device)
    rows, k = a.shape
    if a_scale.numel() != rows:
        raise ValueError(f"a_scale must have {rows} entries, got {a_scale.numel()}")
    if rows > MAX_EXTENT:
        _too_large("rows", rows)
    return rows, k, device


def int8_matmul(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor, *,
                bias: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16,
                status: torch.Tensor | None = None) -> torch.Tensor:
    """``(a @ b.T) * a_scale[:, None] * b_scale (+ bias)`` for int8 ``a`` [M, K] and
    ``b`` [N, K], fp32 scales per row and per output channel and fp32 ``bias``
    [N]. The sum is exact in int32; the result is rounded once to ``out_dtype``.
    ``status`` [1] int32 (zeroed by the caller) gets bit 0 if a bounded wait of
    the kernel ran out, in which case the output is wrong."""
    rows, k, device = _check_rows(a, a_scale)
    _, n = _check_weight("b", b, b_scale, 2, device, k)
    _check_bias(bias, n, device)
    _check_out(out_dtype, status, device)
    args = (a, a_scale, b, b_scale, bias, None, (rows, k, 1, n), out_dtype, 0, status)
    if _differentiated(a_scale, b_scale, bias):
        return _NoGradient.apply("int8_matmul", lambda: _product(*args), a_scale, b_scale, bias)
    return _product(*args)


def int8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                bias: torch.Tensor | None = None, *, out_dtype: torch.dtype | None = None,
                status: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`int8_matmul` of the rows of ``x`` [M, K] (bf16, fp16 or fp32)
    quantised as :func:`quantize_int8` does, in one call; the result has the
    type of ``x`` unless ``out_dtype`` is given."""
    _tensor("x", x, 2, _FLOATS, contiguous=False)
    (rows, k), device = x.shape, x.device
    if rows > MAX_EXTENT:
        _too_large("rows", rows)
    _, n = _check_weight("weight", weight, weight_scale, 2, device, k)
    _check_bias(bias, n, device)
    out_dtype = out_dtype or x.dtype
    _check_out(out_dtype, status, device)
    args = (x, None, weight, weight_scale, bias, None, (rows, k, 1, n), out_dtype, 0, status)
    if _differentiated(x, weight_scale, bias):
        return _NoGradient.apply("int8_linear", lambda: _product(*args), x, weight_scale, bias)
    return _product(*args)


def int8_grouped_matmul(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
                        offsets: torch.Tensor, *, out_dtype: torch.dtype = torch.bfloat16,
                        activation: str | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """Rows ``offsets[g] .. offsets[g + 1]`` of int8 ``a`` [P, K] times ``b[g]`` of
    [G, N, K], scaled as in :func:`int8_matmul` by ``a_scale`` [P] and ``b_scale``
    [G, N]. ``offsets`` [G + 1] int32 ascend (those of :func:`sort_tokens`, from
    0); rows before ``offsets[0]`` and from ``offsets[G]`` on are zeros.
    ``activation="silu_mul"``: the first N / 2 channels are gates, and the
    result [P, N / 2] is silu(gate) * up."""
    rows, k, device = _check_rows(a, a_scale)
    groups, n = _check_weight("b", b, b_scale, 3, device, k)
    _tensor("offsets", offsets, 1, _I32, device)
    if groups > 1024:
        raise ValueError(f"at most 1024 groups are supported, got {groups}")
    if offsets.numel() != groups + 1:
        raise ValueError(f"offsets must have {groups + 1} entries, got {offsets.numel()}")
    if activation not in (None, "silu_mul"):
        raise ValueError(f'activation must be None or "silu_mul", got {activation!r}')
    if activation and n % 2:
        raise ValueError(f"silu_mul needs an even number of channels, got {n}")
    _check_out(out_dtype, status, device)
    args = (a, a_scale, b, b_scale, None, offsets, (rows, k, groups, n), out_dtype, _SILU_MUL if activation else 0, status)
    if _differentiated(a_scale, b_scale):
        return _NoGradient.apply("int8_grouped_matmul", lambda: _product(*args), a_scale, b_scale)
    return _product(*args)


# ---------------------------------------------------------------------------
# the layer
# ---------------------------------------------------------------------------
@lru_cache(maxsize=4096)
def _layer_workspace(m, h, i, e, k, dtype, logits, x_off, w13_off, w2_off) -> int:
    args = _lib.MtpW8A8LayerArgs(m, h, i, e, k, 0, dtype, 0, 256 + x_off, 256 if logits else None, None, None, None,
                                 256 + w13_off, None, 256 + w2_off, None, None, None, None, 0)
    out = _lib.i64()
    _lib.call("mtp_w8a8_moe_layer_workspace_size", C.byref(args), C.byref(out))
    return out.value


def moe_layer_w8a8(hidden_states: torch.Tensor, router_logits: torch.Tensor | None, w13: torch.Tensor,
                   w13_scale: torch.Tensor, w2: torch.Tensor, w2_scale: torch.Tensor, top_k: int,
                   renormalize: bool = True, *, topk_weights: torch.Tensor | None = None,
                   topk_ids: torch.Tensor | None = None, expert_map: torch.Tensor | None = None,
                   out: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """One W8A8 MoE layer forward: router (when ``router_logits`` [M, E] fp32 is
    given, else the given ``topk_weights`` fp32 / ``topk_ids`` int32 [M, k]),
    rows quantised and sorted by expert, ``silu(gate) * up`` of the w13 product
    in fp32, quantised per row, the w2 product, and the weighted sum per token.

    ``hidden_states`` [M, H] bf16, fp16 or fp32; ``w13`` [E, 2I, H] int8 (gate
    rows, then up rows) with ``w13_scale`` [E, 2I]; ``w2`` [E, H, I] int8 with
    ``w2_scale`` [E, H]. Ids outside [0, E) - after ``expert_map``, which takes
    global ids to local ones - contribute nothing. Returns ``out`` [M, H] in
    the type of ``hidden_states`` (a given ``out`` cannot be part of a graph: with
    inputs that require a gradient it raises ``RuntimeError``). ``status`` as in
    :func:`int8_matmul`."""
    _tensor("hidden_states", hidden_states, 2, _FLOATS)
    dev = hidden_states.device
    m, h = hidden_states.shape
    e, n13 = _check_weight("w13", w13, w13_scale, 3, dev, h)
    i = n13 // 2
    if n13 != 2 * i:
        raise ValueError(f"w13 must have gate and up rows, got {n13}")
    if _check_weight("w2", w2, w2_scale, 3, dev, i) != (e, h):
        raise ValueError(f"w2 must be {(e, h, i)}, got {tuple(w2.shape)}")
    if e > 1024:
        raise ValueError(f"at most 1024 experts are supported, got {e}")
    if not 1 <= top_k <= 32:
        raise ValueError(f"top_k must be in [1, 32], got {top_k}")
    if m * top_k > MAX_EXTENT:
        _too_large("pairs", m * top_k)
    if router_logits is not None:
        _tensor("router_logits", router_logits, 2, _F32, dev)
        if router_logits.shape != (m, e):
            raise ValueError(f"router_logits must be {(m, e)}, got {tuple(router_logits.shape)}")
        if top_k > e:
            raise ValueError(f"top_k {top_k} exceeds the {e} experts")
        if expert_map is not None:
            raise ValueError("expert_map needs given topk_ids (global ids), not router_logits")
    else:
        if topk_weights is None or topk_ids is None:
            raise ValueError("give router_logits or topk_weights and topk_ids")
        _tensor("topk_weights", topk_weights, 2, _F32, dev)
        _tensor("topk_ids", topk_ids, 2, _I32, dev)
        if topk_weights.shape != (m, top_k) or topk_ids.shape != (m, top_k):
            raise ValueError(f"topk_weights/topk_ids must be {(m, top_k)}")
    if expert_map is not None:
        _check_map(expert_map, dev)
    if out is not None:
        _tensor("out", out, 2, (hidden_states.dtype,), dev)
        if out.shape != (m, h):
            raise ValueError(f"out must be {(m, h)}, got {tuple(out.shape)}")
    _check_out(hidden_states.dtype, status, dev)
    if router_logits is not None:
        topk_weights = topk_ids = None
    args = (hidden_states, router_logits, w13, w13_scale, w2, w2_scale, (m, h, i, e, top_k), renormalize, topk_weights,
            topk_ids, expert_map, out, status)
    floats = (hidden_states, router_logits, topk_weights, w13_scale, w2_scale)
    if _differentiated(*floats):
        if out is not None:
            raise RuntimeError("moe_layer_w8a8 has no gradient: give no out with inputs that require one")
        return _NoGradient.apply("moe_layer_w8a8", lambda: _layer(*args), *floats)
    return _layer(*args)


def _layer(hidden_states, router_logits, w13, w13_scale, w2, w2_scale, shape, renormalize, topk_weights, topk_ids,
           expert_map, out, status):
    device = hidden_states.get_device()
    if device != _current_device():
        with torch.cuda.device(device):
            return _layer(hidden_states, router_logits, w13, w13_scale, w2, w2_scale, shape, renormalize, topk_weights,
                          topk_ids, expert_map, out, status)
    m, h, i, e, top_k = shape
    if out is None:
        out = torch.empty_like(hidden_states)
    given = router_logits is None
    dtype, px, p13, p2 = DTYPES[hidden_states.dtype], hidden_states.data_ptr(), w13.data_ptr(), w2.data_ptr()
    size = _layer_workspace(m, h, i, e, top_k, dtype, not given, px & 255, p13 & 255, p2 & 255)
    ws = w13.new_empty(size)
    args = _lib.MtpW8A8LayerArgs(m, h, i, e, top_k, 1 if renormalize else 0, dtype,
                                 0 if expert_map is None else expert_map.numel(), px,
                                 None if given else router_logits.data_ptr(),
                                 topk_weights.data_ptr() if given else None, topk_ids.data_ptr() if given else None,
                                 None if expert_map is None else expert_map.data_ptr(), p13, w13_scale.data_ptr(), p2,
                                 w2_scale.data_ptr(), out.data_ptr(), None if status is None else status.data_ptr(),
                                 ws.data_ptr(), size)
    _layer_entry(C.byref(args), _stream(device))
    return out

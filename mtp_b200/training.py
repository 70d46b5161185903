"""What a training step of a mixture-of-experts block needs around the token
sort: torch tensors in, C-ABI calls out.

* :func:`route_tokens` - the router: top-k weights and ids as
  :func:`mtp_b200.topk_softmax` has them, with the gradient of the logits, the
  pairs of every expert, the balance loss and the z loss;
* :func:`layer_norm` - rows normalised, with the gradients of rows, weight and
  bias;
* :func:`embed_tokens` - scaled rows of a table by token ids, with the table's
  gradient summed over the tokens of each row.

Between them go :func:`mtp_b200.sort_tokens` and :func:`mtp_b200.unsort_tokens`,
whose ids and weights are those of :func:`route_tokens`. Shape, dtype and device
errors raise ``ValueError`` before any launch; a non-zero C status raises
:class:`mtp_b200.MtpError`. Every call is asynchronous on the current torch
stream of its tensors' GPU, which need not be the current one. There is no CPU
path. Gradients are first derivatives, backward; forward mode raises
``RuntimeError``. All sums are in fp32 or more and in an order that sizes and
memory layout fix, not timing: the same call gives the same bits. (Should a
bounded wait of a layer norm kernel run out, the rows that it was for are NaN,
rows behind them may be, and so may columns of the sums over them.)
"""
from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple

import torch

from . import _lib
from .w8a8 import (DTYPES, MAX_EXTENT, _F32, _FLOATS, _current_device, _differentiated, _given_back, _row_stride, _stream,
                   _tensor, _too_large)

_MOST = torch.finfo(torch.float32).max
_PARAMS = {t: _F32 if t == torch.float32 else (t, torch.float32) for t in _FLOATS}  # types of a layer norm's parameters

_route_entry = _lib.Entry("mtp_route_tokens")
_route_backward_entry = _lib.Entry("mtp_route_tokens_backward")
_norm_entry = _lib.Entry("mtp_layer_norm")
_norm_backward_entry = _lib.Entry("mtp_layer_norm_backward")
_embed_entry = _lib.Entry("mtp_embed_tokens")
_embed_backward_entry = _lib.Entry("mtp_embed_tokens_backward")


@lru_cache(maxsize=4096)
def _workspace(name: str, *shape) -> int:
    out = _lib.i64()
    _lib.call(name, *shape, _lib.C.byref(out))
    return out.value


def _ptr(t):
    return None if t is None else t.data_ptr()


def _like(x):
    """A contiguous tensor as x; empty_like is the cheapest of torch's calls, and keeps the strides of a slice's rows."""
    return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


def _is_row(t, index, dtypes, n) -> bool:
    """What _tensor and a check of the size ask of a contiguous t [n], in the order of a call that is right."""
    return (isinstance(t, torch.Tensor) and t.get_device() == index and t.dtype in dtypes and t.ndim == 1
            and t.shape[0] == n and t.is_contiguous())


def _first_derivative(backward):
    """A backward pass whose own derivative is an error. Outside create_graph nothing records one, and
    once_differentiable's detour (9 us of the 75 that a small layer norm's backward pass takes) is left out."""
    checked = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        return (checked if torch.is_grad_enabled() else backward)(ctx, *grads)

    return staticmethod(run)


# ---------------------------------------------------------------------------
# router
# ---------------------------------------------------------------------------
class RoutedTokens(NamedTuple):
    """What :func:`route_tokens` returns.

    ``weights`` [M, k] fp32 and ``ids`` [M, k] int32 (0 and -1 for a token that
    does not count), ``counts`` [E] int32 pairs of each expert,
    ``balance_loss`` and ``z_loss``, fp32 numbers."""

    weights: torch.Tensor
    ids: torch.Tensor
    counts: torch.Tensor
    balance_loss: torch.Tensor
    z_loss: torch.Tensor


def _route(logits, stride, top_k, renormalize, token_mask, need_pull):
    device = logits.get_device()
    if device != _current_device():
        with torch.cuda.device(device):
            return _route(logits, stride, top_k, renormalize, token_mask, need_pull)
    m, e = logits.shape
    weights = logits.new_empty(m, top_k, dtype=torch.float32)
    ids = logits.new_empty(m, top_k, dtype=torch.int32)
    counts = logits.new_empty(e, dtype=torch.int32)
    balance = logits.new_empty((), dtype=torch.float32)
    z = logits.new_empty((), dtype=torch.float32)
    pull = logits.new_empty(e + 1, dtype=torch.float32) if need_pull else None
    size = _workspace("mtp_route_tokens_workspace_size", m, e)
    ws = logits.new_empty(size, dtype=torch.uint8) if size else None
    _route_entry(logits.data_ptr() or None, stride, DTYPES[logits.dtype], m, e, top_k,
                 1 if renormalize else 0, _ptr(token_mask), weights.data_ptr(), ids.data_ptr(), counts.data_ptr(),
                 balance.data_ptr(), z.data_ptr(), _ptr(pull), _ptr(ws), size, _stream(device))
    return weights, ids, counts, balance, z, pull


def _route_backward(logits, stride, top_k, renormalize, token_mask, ids, pull, grad_weights, grad_balance, grad_z):
    device = logits.get_device()
    if device != _current_device():
        with torch.cuda.device(device):
            return _route_backward(logits, stride, top_k, renormalize, token_mask, ids, pull, grad_weights, grad_balance,
                                   grad_z)
    m, e = logits.shape
    grad = logits.new_empty(m, e)
    _route_backward_entry(logits.data_ptr(), stride, DTYPES[logits.dtype], m, e, top_k,
                          1 if renormalize else 0, _ptr(token_mask), ids.data_ptr(), pull.data_ptr(),
                          _ptr(grad_weights), _ptr(grad_balance), _ptr(grad_z), grad.data_ptr(), _stream(device))
    return grad


class _RouteTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, stride, top_k, renormalize, token_mask, rest):
        # ids and counts are not differentiable: they go around autograd, in `rest`
        weights, ids, counts, balance, z, pull = _route(logits, stride, top_k, renormalize, token_mask, True)
        ctx.save_for_backward(logits, ids, pull, token_mask)
        ctx.saved = logits.shape, logits.dtype, logits.device
        ctx.top_k, ctx.renormalize = top_k, renormalize
        ctx.set_materialize_grads(False)
        rest.extend((ids, counts))
        return weights, balance, z

    @_first_derivative
    def backward(ctx, grad_weights, grad_balance, grad_z):
        logits, ids, pull, token_mask = ctx.saved_tensors
        shape, dtype, device = ctx.saved
        (m, e), k = shape, ctx.top_k
        logits = _given_back("router_logits", logits, shape, dtype, device, rows=True)
        ids = _given_back("ids", ids, (m, k), torch.int32, device)
        pull = _given_back("counts' terms", pull, (e + 1,), torch.float32, device)
        if token_mask is not None:
            token_mask = _given_back("token_mask", token_mask, (m,), torch.bool, device)
        if grad_weights is not None:
            grad_weights = grad_weights.contiguous()
        return (_route_backward(logits, _row_stride("router_logits", logits), k, ctx.renormalize, token_mask, ids, pull,
                                grad_weights, grad_balance, grad_z), None, None, None, None, None)


def route_tokens(router_logits: torch.Tensor, top_k: int, renormalize: bool = True, *,
                 token_mask: torch.Tensor | None = None) -> RoutedTokens:
    """The router of a training step for ``router_logits`` [M, E] (bf16, fp16 or
    fp32): p = softmax of a row in fp32, ``ids`` the ``top_k`` largest (ties: the
    lower id), ``weights`` p there, divided by their sum with ``renormalize``.

    Tokens whose ``token_mask`` [M] bool is false do not count: their ids are -1
    and their weights 0, so that :func:`mtp_b200.sort_tokens` gives them no
    expert, and their logits, whatever they hold, get zeros as gradient. Over the
    n tokens that count, ``counts[e]`` are the pairs of expert e,
    ``balance_loss = E / (k n^2) * sum_e counts[e] * sum_t p[t, e]`` (1 where
    experts are used evenly) and ``z_loss = sum_t logsumexp(logits[t])^2 / n``;
    both are 0 for n = 0. Gradients go from ``weights``, ``balance_loss`` (with
    counts as constants) and ``z_loss`` to the logits. A token with a NaN or a
    positive infinity has NaN weights, distinct ids, and makes both losses NaN."""
    _tensor("router_logits", router_logits, 2, _FLOATS, contiguous=False)
    m, e = router_logits.shape
    if not 1 <= e <= 1024:
        raise ValueError(f"1 to 1024 experts are supported, got {e}")
    if not 1 <= top_k <= min(e, 32):
        raise ValueError(f"top_k must be in [1, {min(e, 32)}], got {top_k}")
    if m * top_k > MAX_EXTENT:
        _too_large("pairs", m * top_k)
    stride = _row_stride("router_logits", router_logits)
    if token_mask is not None:
        _tensor("token_mask", token_mask, 1, (torch.bool,), router_logits.device)
        if token_mask.numel() != m:
            raise ValueError(f"token_mask must have {m} entries, got {token_mask.numel()}")
    if _differentiated(router_logits):
        rest = []
        weights, balance, z = _RouteTokens.apply(router_logits, stride, top_k, renormalize, token_mask, rest)
        return RoutedTokens(weights, *rest, balance, z)
    return RoutedTokens(*_route(router_logits, stride, top_k, renormalize, token_mask, False)[:5])


# ---------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------
def _rows_of(x):
    """(rows, elements between them) of a tensor whose last dimension is normalised."""
    if x.ndim == 2:
        return x.shape[0], _row_stride("x", x)
    return x.numel() // x.shape[-1], x.shape[-1]


def _norm(x, rows, weight, bias, eps, need_stats):
    device = x.get_device()
    if device != _current_device():
        with torch.cuda.device(device):
            return _norm(x, rows, weight, bias, eps, need_stats)
    (m, stride), h = rows, x.shape[-1]
    y = _like(x)
    stats = x.new_empty(m, 2, dtype=torch.float32) if need_stats else None
    param = x.dtype if weight is None and bias is None else (bias if weight is None else weight).dtype
    _norm_entry(x.data_ptr(), stride, DTYPES[x.dtype], m, h, _ptr(weight), _ptr(bias), DTYPES[param], eps,
                y.data_ptr(), _ptr(stats), _stream(device))
    return y, stats


def _norm_backward(grad, x, rows, weight, stats, param, need_x, need_weight, need_bias):
    device = x.get_device()
    if device != _current_device():
        with torch.cuda.device(device):
            return _norm_backward(grad, x, rows, weight, stats, param, need_x, need_weight, need_bias)
    (m, stride), h = rows, x.shape[-1]
    grad_x = _like(x) if need_x else None
    grad_weight = torch.empty_like(weight) if need_weight else None
    grad_bias = x.new_empty(h, dtype=param) if need_bias else None
    size = _workspace("mtp_layer_norm_backward_workspace_size", m, h) if need_weight or need_bias else 0
    ws = x.new_empty(size, dtype=torch.uint8) if size else None
    _norm_backward_entry(grad.data_ptr(), x.data_ptr(), stride, DTYPES[x.dtype], m, h, _ptr(weight), DTYPES[param],
                         stats.data_ptr(), _ptr(grad_x), _ptr(grad_weight), _ptr(grad_bias), _ptr(ws), size,
                         _stream(device))
    return grad_x, grad_weight, grad_bias


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, rows, weight, bias, eps):
        y, stats = _norm(x, rows, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.param = x.dtype if weight is None and bias is None else (bias if weight is None else weight).dtype
        return y

    @_first_derivative
    def backward(ctx, grad):
        x, weight, stats = ctx.saved_tensors
        need_x, _, need_weight, need_bias, _ = ctx.needs_input_grad
        device, h = grad.device, grad.shape[-1]
        x = _given_back("x", x, grad.shape, grad.dtype, device, rows=True)
        rows = _rows_of(x)
        stats = _given_back("rows' statistics", stats, (rows[0], 2), torch.float32, device)
        if weight is not None:
            weight = _given_back("weight", weight, (h,), ctx.param, device)
        grad_x, grad_weight, grad_bias = _norm_backward(grad.contiguous(), x, rows, weight, stats, ctx.param, need_x,
                                                        need_weight, need_bias)
        return grad_x, None, grad_weight, grad_bias, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension H of
    ``x`` [..., H] (bf16, fp16 or fp32; a 2-D ``x`` may be a slice of wider rows),
    in fp32 and rounded once to the type of ``x``. ``weight`` and ``bias`` [H]
    (None: 1 and 0) have the type of ``x`` or are both fp32. Gradients go to all
    three; those of ``weight`` and ``bias`` are summed over the rows in fp32 and
    rounded once."""
    if not isinstance(x, torch.Tensor):
        raise TypeError("x must be a torch.Tensor")
    if x.ndim < 1:
        raise ValueError("x must have at least one dimension")
    _tensor("x", x, x.ndim, _FLOATS, contiguous=x.ndim != 2)
    h = x.shape[-1]
    if h < 1:
        raise ValueError("x must have at least one column")
    if h > MAX_EXTENT:
        _too_large("columns", h)
    if x.numel() // h > MAX_EXTENT:
        _too_large("rows", x.numel() // h)
    rows = _rows_of(x)
    types, index = _PARAMS[x.dtype], x.get_device()
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and not _is_row(t, index, types, h):
            _tensor(name, t, 1, types, x.device)
            raise ValueError(f"{name} must have {h} entries, got {t.numel()}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"weight and bias must have one type, got {weight.dtype} and {bias.dtype}")
    if not 0 <= eps <= _MOST:
        raise ValueError(f"eps must be a number of fp32 from 0 on, got {eps}")
    if _differentiated(x, weight, bias):
        return _LayerNorm.apply(x, rows, weight, bias, eps)
    return _norm(x, rows, weight, bias, eps, False)[0]


# ---------------------------------------------------------------------------
# embedding
# ---------------------------------------------------------------------------
def _embed(ids, table, scale):
    device = table.get_device()
    if device != _current_device():
        with torch.cuda.device(device):
            return _embed(ids, table, scale)
    v, h = table.shape
    out = table.new_empty(*ids.shape, h)
    _embed_entry(ids.data_ptr(), ids.element_size(), ids.numel(), table.data_ptr(), DTYPES[table.dtype], v, h, scale,
                 out.data_ptr(), _stream(device))
    return out


def _embed_backward(ids, grad, v, scale):
    device = grad.get_device()
    if device != _current_device():
        with torch.cuda.device(device):
            return _embed_backward(ids, grad, v, scale)
    n, h, dtype = ids.numel(), grad.shape[-1], DTYPES[grad.dtype]
    grad_table = grad.new_empty(v, h)
    size = _workspace("mtp_embed_tokens_backward_workspace_size", n, h, dtype)
    ws = grad.new_empty(size, dtype=torch.uint8)
    _embed_backward_entry(ids.data_ptr() or None, ids.element_size(), n, grad.data_ptr() or None, dtype, v, h, scale,
                          grad_table.data_ptr(), ws.data_ptr(), size, _stream(device))
    return grad_table


class _EmbedTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale):
        ctx.save_for_backward(ids)
        ctx.v, ctx.scale, ctx.id_type = table.shape[0], scale, ids.dtype
        return _embed(ids, table, scale)

    @_first_derivative
    def backward(ctx, grad):
        (ids,) = ctx.saved_tensors
        ids = _given_back("ids", ids, grad.shape[:-1], ctx.id_type, grad.device)
        return None, _embed_backward(ids, grad.contiguous(), ctx.v, ctx.scale), None


def embed_tokens(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """``scale * table[ids]`` [..., H] for ``ids`` [...] int32 or int64 and a
    ``table`` [V, H] (bf16, fp16 or fp32), in fp32 and rounded once. An id outside
    [0, V) - padding, or a row of another rank's part of the table - gives zeros.
    The gradient of ``table`` [V, H] sums the gradients of each row's tokens,
    ascending, in fp32, times ``scale``, rounded once; rows without a token get
    zeros."""
    if not isinstance(ids, torch.Tensor):
        raise TypeError("ids must be a torch.Tensor")
    _tensor("table", table, 2, _FLOATS)
    _tensor("ids", ids, ids.ndim, (torch.int32, torch.int64), table.device)
    v, h = table.shape
    if not v or not h:
        raise ValueError(f"table must not be empty, got shape {tuple(table.shape)}")
    for what, n in (("ids", ids.numel()), ("rows of table", v), ("columns", h)):
        if n > MAX_EXTENT:
            _too_large(what, n)
    if not isinstance(scale, (int, float)) or not abs(scale) <= _MOST:
        raise ValueError(f"scale must be a finite number of fp32, got {scale!r}")
    if _differentiated(table):
        return _EmbedTokens.apply(ids, table, scale)
    return _embed(ids, table, scale)

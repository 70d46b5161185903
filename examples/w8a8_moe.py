"""The int8 (W8A8) expert path as a model uses it, on one GPU.

    python examples/w8a8_moe.py [--tokens 512] [--hidden 2048] [--inter 512] [--experts 64] [--top-k 8]

Serving: the experts' weights are quantised once (one scale per output channel),
then a layer call is the routed experts (``moe_layer_w8a8``) plus a sigmoid-gated
shared expert whose two projections are ``int8_linear``. The result is compared
with the same layer on the unquantised weights.

Training: the router and the experts of such a layer learn to imitate a teacher;
the tokens go to their experts and back through ``route_tokens``, ``sort_tokens``
and ``unsort_tokens``, whose gradients reach the logits, the rows and the routing
weights.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import mtp_b200  # noqa: E402


def quantize_channels(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """int8 codes and one fp32 scale per output channel of weights [..., out, in]."""
    codes, scale = mtp_b200.quantize_int8(w.flatten(0, -2).contiguous())
    return codes.contiguous().view(w.shape), scale.view(w.shape[:-1])


class W8A8Layer:
    """Router, routed experts and gated shared expert with int8 weights."""

    def __init__(self, router, w13, w2, shared13, shared2, shared_gate, top_k):
        self.router, self.shared_gate, self.top_k = router, shared_gate, top_k
        self.w13, self.w2 = quantize_channels(w13), quantize_channels(w2)
        self.shared13, self.shared2 = quantize_channels(shared13), quantize_channels(shared2)

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        logits = (x @ self.router.T).float()
        routed = mtp_b200.moe_layer_w8a8(x, logits, *self.w13, *self.w2, self.top_k)
        gate, up = mtp_b200.int8_linear(x, *self.shared13).chunk(2, -1)
        shared = mtp_b200.int8_linear((torch.nn.functional.silu(gate) * up).contiguous(), *self.shared2)
        return routed + torch.sigmoid(x @ self.shared_gate)[:, None] * shared


def plain_layer(x, router, w13, w2, shared13, shared2, shared_gate, top_k):
    """The same layer on the weights as they are, in fp32."""
    def expert(rows, a, b):
        gate, up = (rows @ a.float().T).chunk(2, -1)
        return (torch.nn.functional.silu(gate) * up) @ b.float().T

    weights, ids, _ = mtp_b200.topk_softmax((x @ router.T).float(), top_k)
    out, rows = torch.zeros_like(x, dtype=torch.float32), x.float()
    for e in range(w13.shape[0]):
        t, j = (ids == e).nonzero(as_tuple=True)
        out.index_add_(0, t, expert(rows[t], w13[e], w2[e]) * weights[t, j, None])
    return out + torch.sigmoid(x @ shared_gate).float()[:, None] * expert(rows, shared13, shared2)


def serve(args, g) -> float:
    def normal(*shape):
        return (torch.randn(*shape, generator=g, device="cuda") / shape[-1] ** 0.5).to(torch.bfloat16)

    h, i, e = args.hidden, args.inter, args.experts
    weights = (normal(e, h), normal(e, 2 * i, h), normal(e, h, i), normal(2 * i, h), normal(h, i), normal(h), args.top_k)
    layer = W8A8Layer(*weights)
    worst = 0.0
    for tokens in sorted({1, args.tokens}):
        x = torch.randn(tokens, h, generator=g, device="cuda").to(torch.bfloat16)
        out, ref = layer(x).float(), plain_layer(x, *weights)
        error = float((out - ref).norm() / ref.norm())
        worst = max(worst, error)
        print(f"serving {tokens:5d} tokens: relative error of the int8 layer {error:.4f}")
    return worst


def train(args, g) -> tuple[float, float]:
    """First and last loss of a few steps on one batch."""
    h, e, k, m = args.hidden, args.experts, args.top_k, args.tokens
    scale = h ** -0.5
    x = torch.randn(m, h, generator=g, device="cuda")
    target = torch.tanh(x @ (torch.randn(h, h, generator=g, device="cuda") * scale))
    router = (torch.randn(e, h, generator=g, device="cuda") * scale).requires_grad_()
    experts = (torch.randn(e, h, h, generator=g, device="cuda") * scale).requires_grad_()
    optimizer = torch.optim.Adam([router, experts], lr=1e-3)
    losses = []
    for _ in range(args.steps):
        logits = x @ router.T
        weights, ids, *_ = mtp_b200.route_tokens(logits, k)
        rows, positions, offsets, _ = mtp_b200.sort_tokens(x, ids, e)
        ends = offsets.tolist()
        y = torch.cat([rows[ends[n]:ends[n + 1]] @ experts[n].T for n in range(e)])
        loss = (mtp_b200.unsort_tokens(y, positions, weights) - target).square().mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
    print(f"training {args.steps} steps: loss {losses[0]:.4f} -> {losses[-1]:.4f}")
    return losses[0], losses[-1]


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("tokens", 512), ("hidden", 2048), ("inter", 512), ("experts", 64), ("top-k", 8), ("steps", 10)):
        ap.add_argument(f"--{name}", type=int, default=value)
    args = ap.parse_args(argv)
    g = torch.Generator(device="cuda").manual_seed(0)
    return serve(args, g), train(args, g)


if __name__ == "__main__":
    main()

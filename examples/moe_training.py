"""A mixture-of-experts block in training, from token ids to its gradients, on one GPU.

    python examples/moe_training.py [--tokens 2048] [--hidden 512] [--experts 16] [--top-k 2] [--vocabulary 4096] [--steps 10]

Token ids (some of them padding) go through ``embed_tokens``, ``layer_norm``, ``route_tokens``, ``sort_tokens``, one
matrix per expert, and ``unsort_tokens``; the loss is the distance to a teacher plus the router's balance and z losses.
The gradients of the first step are compared with the same block in plain torch operations.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import mtp_b200  # noqa: E402

BALANCE, Z_LOSS = 0.01, 0.001


class Block:
    def __init__(self, args, g):
        def normal(*shape):
            return torch.randn(*shape, generator=g, device="cuda")

        h, e = args.hidden, args.experts
        self.top_k, self.scale = args.top_k, h ** 0.5
        self.table = normal(args.vocabulary, h) / self.scale
        self.weight, self.bias = torch.ones(h, device="cuda"), torch.zeros(h, device="cuda")
        self.router, self.experts = normal(e, h) / self.scale, normal(e, h, h) / self.scale
        for p in self.parameters():
            p.requires_grad_()

    def parameters(self):
        return [self.table, self.weight, self.bias, self.router, self.experts]

    def loss(self, ids, target):
        """(loss, distance to the target, balance loss); tokens with a negative id are padding."""
        x = mtp_b200.layer_norm(mtp_b200.embed_tokens(ids, self.table, self.scale), self.weight, self.bias)
        r = mtp_b200.route_tokens(x @ self.router.T, self.top_k, token_mask=ids >= 0)
        rows, positions, offsets, _ = mtp_b200.sort_tokens(x, r.ids, len(self.experts))
        ends = offsets.tolist()
        parts = [rows[ends[n]:ends[n + 1]] @ w.T for n, w in enumerate(self.experts)]
        parts.append(rows.new_zeros(len(rows) - ends[-1], rows.shape[1]))  # the padding's rows
        y = mtp_b200.unsort_tokens(torch.cat(parts), positions, r.weights)
        distance = (y - target).square().mean()
        return distance + BALANCE * r.balance_loss + Z_LOSS * r.z_loss, distance, r.balance_loss

    def plain_loss(self, ids, target):
        """The same in plain torch operations."""
        real = ids >= 0
        x = torch.where(real[:, None], self.table[ids.long().clamp(min=0)] * self.scale, 0.0)
        x = torch.nn.functional.layer_norm(x, x.shape[-1:], self.weight, self.bias)
        logits = x @ self.router.T
        p = torch.softmax(logits, -1)
        chosen = torch.topk(logits.detach(), self.top_k, -1).indices
        w = p.gather(1, chosen)
        w = w / w.sum(-1, keepdim=True) * real[:, None]
        y = torch.zeros_like(x)
        for n, expert in enumerate(self.experts):
            t, j = (chosen == n).nonzero(as_tuple=True)
            y = y.index_add(0, t, (x[t] @ expert.T) * w[t, j, None])
        n = real.sum()
        counts = torch.bincount(chosen[real].flatten(), minlength=len(self.experts))
        balance = len(self.experts) / (self.top_k * n * n) * (counts * p[real].sum(0)).sum()
        return (y - target).square().mean() + BALANCE * balance + Z_LOSS * torch.logsumexp(logits[real], -1).square().mean()


def main(argv=None) -> dict[str, float]:
    """The relative difference of each parameter's gradient from plain torch's."""
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("tokens", 2048), ("hidden", 512), ("experts", 16), ("top-k", 2), ("vocabulary", 4096), ("steps", 10)):
        ap.add_argument(f"--{name}", type=int, default=value)
    args = ap.parse_args(argv)
    g = torch.Generator(device="cuda").manual_seed(0)
    block = Block(args, g)
    ids = torch.randint(0, args.vocabulary, (args.tokens,), generator=g, device="cuda", dtype=torch.int32)
    ids[-args.tokens // 8:] = -1
    target = torch.tanh(torch.randn(args.tokens, args.hidden, generator=g, device="cuda"))

    names = ("table", "weight", "bias", "router", "experts")
    ours = torch.autograd.grad(block.loss(ids, target)[0], block.parameters())
    plain = torch.autograd.grad(block.plain_loss(ids, target), block.parameters())
    difference = {n: float((a - b).norm() / b.norm()) for n, a, b in zip(names, ours, plain)}
    print("gradients against plain torch:", ", ".join(f"{n} {d:.1e}" for n, d in difference.items()))

    optimizer = torch.optim.Adam(block.parameters(), lr=1e-3)
    for step in range(args.steps):
        loss, distance, balance = block.loss(ids, target)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        print(f"step {step}: loss {loss.item():.4f}, distance {distance.item():.4f}, balance {balance.item():.3f}")
    return difference


if __name__ == "__main__":
    main()

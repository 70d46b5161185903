"""The operators of a training step as they are used together: a block from token ids to a loss against 64 bits, on
another stream, two streams at once, and captured into a graph."""
import pytest
import torch

pytestmark = pytest.mark.gpu

I32 = torch.int32


class Block:
    """embedding -> layer norm -> router -> sort -> experts -> unsort -> loss."""

    def __init__(self, v=300, h=64, e=6, k=2, m=200, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        n = lambda *s: torch.randn(*s, generator=g, device="cuda")
        self.k, self.e = k, e
        self.table, self.w, self.b = n(v, h) / 8, 1 + 0.1 * n(h), 0.1 * n(h)
        self.router, self.experts = n(e, h) / 8, n(e, h, h) / 8
        self.ids = torch.randint(-1, v, (m,), generator=g, device="cuda", dtype=I32)
        self.mask = self.ids >= 0
        self.target = n(m, h)
        self.leaves = [self.table, self.w, self.b, self.router, self.experts]
        for t in self.leaves:
            t.requires_grad_()

    def loss(self):
        import mtp_b200
        x = mtp_b200.layer_norm(mtp_b200.embed_tokens(self.ids, self.table, 8.0), self.w, self.b)
        r = mtp_b200.route_tokens(x @ self.router.T, self.k, token_mask=self.mask)
        rows, positions, offsets, _ = mtp_b200.sort_tokens(x, r.ids, self.e)
        # every row times its expert's matrix, without a look at the offsets on the host
        at = torch.arange(rows.shape[0], device="cuda")
        expert = torch.searchsorted(offsets[1:].contiguous(), at, right=True)
        weight = torch.cat([self.experts, torch.zeros_like(self.experts[:1])])[expert]
        y = torch.bmm(weight, rows[..., None])[..., 0]
        out = mtp_b200.unsort_tokens(y, positions, r.weights)
        self.ids_chosen = r.ids
        return (out - self.target).square().mean() + 0.01 * r.balance_loss + 0.001 * r.z_loss

    def grads(self):
        loss = self.loss()
        return (loss.detach(), *torch.autograd.grad(loss, self.leaves))

    def exact(self):
        """The same in 64 bits with torch alone, for the experts that were chosen."""
        leaves = [t.detach().double().requires_grad_() for t in self.leaves]
        table, w, b, router, experts = leaves
        x = torch.where(self.mask[:, None], 8.0 * table[self.ids.long().clamp(min=0)], 0.0)
        x = (x - x.mean(-1, keepdim=True)) / (x.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt() * w + b
        z = x @ router.T
        p = torch.softmax(z, -1)
        ids = self.ids_chosen.long().clamp(min=0)
        pw = p.gather(1, ids)
        pw = pw / pw.sum(-1, keepdim=True) * self.mask[:, None]
        y = torch.einsum("mkij,mj->mki", experts[ids], x)
        out = (y * pw[..., None]).sum(1)
        n = self.mask.sum()
        counts = torch.bincount(ids[self.mask].flatten(), minlength=self.e).double()
        balance = self.e / (self.k * n * n) * (counts @ p[self.mask].sum(0))
        z_loss = torch.logsumexp(z[self.mask], -1).square().mean()
        loss = (out - self.target).square().mean() + 0.01 * balance + 0.001 * z_loss
        return (loss.detach(), *torch.autograd.grad(loss, leaves))


def close(got, want):
    # eight steps there and back, each within 2^-17 of its result's norm (sums of at most 200 products in fp32: 200 u =
    # 2^-16.4 at worst), whose errors pass through factors of about one
    for x, y in zip(got, want):
        assert float((x.double() - y).norm()) <= 2.0 ** -12 * float(y.norm()), (float((x.double() - y).norm()), float(y.norm()))


@pytest.fixture(autouse=True)
def no_tf32():
    before = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    yield
    torch.backends.cuda.matmul.allow_tf32 = before


@pytest.mark.parametrize("m", [1, 30, 700])
def test_block_and_its_gradients(cuda_device, m):
    block = Block(m=m, seed=m)
    if m == 1:
        block.ids.fill_(5)
        block.mask.fill_(True)
    got = block.grads()
    close(got, block.exact())


def test_on_another_stream(cuda_device):
    """Inputs made on a side stream just before the calls, results read on it."""
    want = Block(seed=3).grads()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        block = Block(seed=3)
        keep = [t.detach().clone() for t in block.leaves]
        with torch.no_grad():
            for t in block.leaves:
                t.fill_(float("nan"))
            torch.cuda._sleep(20_000_000)
            for t, k in zip(block.leaves, keep):
                t.copy_(k)
        got = block.grads()
    side.synchronize()
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_two_streams_at_once(cuda_device):
    blocks = [Block(m=3000, v=5000, seed=s) for s in (1, 2)]
    want = [b.grads() for b in blocks]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in blocks]
    got = [[], []]
    for _ in range(4):
        for i, (s, b) in enumerate(zip(streams, blocks)):
            with torch.cuda.stream(s):
                got[i].append(b.grads())
    torch.cuda.synchronize()
    for w, gs in zip(want, got):
        for g in gs:
            for x, y in zip(g, w):
                assert torch.equal(x, y)


def test_captured_and_replayed(cuda_device):
    """Forward and backward in one graph: replays on other inputs, two graphs one after the other."""
    want, blocks, graphs, outs = [], [], [], []
    for seed in (11, 12):
        want.append(Block(seed=seed, m=500).grads())
    torch.cuda.synchronize()
    for _ in range(2):
        block = Block(seed=10, m=500)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            block.grads()  # loads the kernels
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = block.grads()
        blocks.append(block)
        graphs.append(graph)
        outs.append(out)
    for turn in range(3):
        for i in (0, 1):
            other = Block(seed=11 + (i + turn) % 2, m=500)
            with torch.no_grad():
                for t, k in zip(blocks[i].leaves, other.leaves):
                    t.copy_(k)
            blocks[i].ids.copy_(other.ids)
            blocks[i].mask.copy_(other.mask)
            blocks[i].target.copy_(other.target)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            for x, y in zip(outs[i], want[(i + turn) % 2]):
                assert torch.equal(x, y)


def test_gradients_add_up_over_two_calls(cuda_device):
    """One table and one router used twice in a step."""
    import mtp_b200
    block = Block()
    once = block.grads()
    loss = block.loss() + block.loss()
    for x, y in zip(torch.autograd.grad(loss, block.leaves), once[1:]):
        assert torch.equal(x, 2 * y)
    block.table.grad = None
    mtp_b200.embed_tokens(block.ids, block.table).sum().backward()
    first = block.table.grad.clone()
    mtp_b200.embed_tokens(block.ids, block.table).sum().backward()
    assert torch.equal(block.table.grad, 2 * first)


def test_backward_into_grads_captured(cuda_device):
    """loss.backward() in a graph, with no eager graph of the same leaves alive: the gradients it leaves in .grad."""
    import gc
    want = Block(seed=5, m=400).grads()
    block = Block(seed=5, m=400)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block.loss().backward()  # loads the kernels
    torch.cuda.current_stream().wait_stream(side)
    for t in block.leaves:
        t.grad = None
    gc.collect()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = block.loss()
        loss.backward()
    for t in block.leaves:
        t.grad.fill_(float("nan"))
    graph.replay()
    torch.cuda.synchronize()
    for x, y in zip((loss.detach(), *(t.grad for t in block.leaves)), want):
        assert torch.equal(x, y)


@pytest.mark.parametrize("order", [0, 1])
def test_calls_of_other_sizes_between(cuda_device, order):
    """Nothing of one call is left for the next: a small step between two large ones, and the other way round."""
    sizes = [(3000, 5000), (7, 20)] if order else [(7, 20), (3000, 5000)]
    blocks = [Block(m=m, v=v, seed=m) for m, v in sizes]
    first = [b.grads() for b in blocks]
    for _ in range(2):
        for b, w in zip(blocks, first):
            for x, y in zip(b.grads(), w):
                assert torch.equal(x, y)

"""Cases of the operators around the token sort in a training step of a mixture-of-experts block.

Three operators, each a public call of ``mtp_b200``:

* ``route`` - ``route_tokens``: softmax, top-k and renormalised weights of the router's logits, the
              pairs of every expert, the balance loss and the z loss, and the gradient of the logits;
* ``norm``  - ``layer_norm``: rows normalised, and the gradients of rows, weight and bias;
* ``embed`` - ``embed_tokens``: scaled rows of a table, and the table's gradient summed over the
              tokens of every row.

``run`` computes them in elementary torch operations where ``own`` is false and through the package
where it is true.

Definitions. ``route``, for n counted tokens (all, or those whose mask is true): p = softmax(z),
ids = the k largest (ties: lowest id), w = p[ids], divided by their sum where renormalised; a token
that does not count has ids -1 and weights 0. counts[e] = pairs of e, balance = E / (k n^2) *
sum_e counts[e] * sum_t p[t, e], z_loss = sum_t logsumexp(z[t])^2 / n. ``norm``: y = (x - mean) /
sqrt(var + eps) * w + b. ``embed``: out = scale * table[id]; an id outside the table gives zeros.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-5
BALANCE, Z_LOSS = 0.01, 0.001  # the losses' weights in a training step

# The largest listed cases bound what a drawn one may cost.
MOST_LOGITS = 65536 * 512
MOST_ACTIVATIONS = 16384 * 8192
MOST_TABLE = 131072 * 2048
MOST_LOOKED_UP = 65536 * 2048


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one decode token, 256 experts, top-8: all latency
        dict(name="route, one token", op="route", m=1, e=256, k=8, dtype="fp32", renorm=True, mask=False, train=False),
        # a training step's chunk: weights, counts, both losses and the gradient of the logits
        dict(name="route, training chunk", op="route", m=8192, e=256, k=8, dtype="fp32", renorm=True, mask=False, train=True),
        # a padded batch with odd sizes, 16-bit logits and weights that are not renormalised
        dict(name="route, padded batch", op="route", m=3001, e=60, k=6, dtype="bf16", renorm=False, mask=True, train=True),
        # the tokens of a long step over many experts
        dict(name="route, long step", op="route", m=65536, e=512, k=8, dtype="fp32", renorm=True, mask=False, train=True),
        # one decode token
        dict(name="norm, one token", op="norm", m=1, h=2048, dtype="bf16", params="bf16", affine=True, strided=False, train=False),
        # a training step's chunk, 16-bit rows and fp32 parameters
        dict(name="norm, training chunk", op="norm", m=8192, h=2048, dtype="bf16", params="fp32", affine=True, strided=False, train=True),
        # odd sizes, fp32, rows that are a part of wider ones
        dict(name="norm, odd rows", op="norm", m=1531, h=1001, dtype="fp32", params="fp32", affine=True, strided=True, train=True),
        # a long step of a wide model
        dict(name="norm, wide rows", op="norm", m=16384, h=8192, dtype="bf16", params="bf16", affine=True, strided=False, train=True),
        # one decode token's row of the vocabulary
        dict(name="embed, one token", op="embed", n=1, v=131072, h=2048, dtype="bf16", padding=False, train=False),
        # a training step's chunk: rows out, the whole vocabulary's gradient back
        dict(name="embed, training chunk", op="embed", n=8192, v=131072, h=2048, dtype="bf16", padding=False, train=True),
        # the predictor's table of layers: every row belongs to many tokens
        dict(name="embed, layer table", op="embed", n=8192, v=40, h=2048, dtype="fp32", padding=False, train=True),
        # a long step with padding, odd sizes
        dict(name="embed, padded step", op="embed", n=61441, v=50021, h=1000, dtype="bf16", padding=True, train=True),
    ]


def _spread(rng, low, high):
    """A whole number in [low, high], even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width(rng, low, high):
    """Three widths in four are multiples of 8, as models have them; the others stay as drawn."""
    h = _spread(rng, low, high)
    return max(8, h // 8 * 8) if rng.random() < 0.75 else h


def draw(rng):
    op = rng.choice(["route", "norm", "embed"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    train = rng.random() < 0.7
    if op == "route":
        e = _spread(rng, 2, 1024)
        m = _spread(rng, 1, min(65536, MOST_LOGITS // e))
        return dict(op=op, m=m, e=e, k=rng.randint(1, min(e, 16)), dtype=rng.choice(["fp32", "fp32", dtype]),
                    renorm=rng.random() < 0.7, mask=rng.random() < 0.4, train=train)
    if op == "norm":
        h = _width(rng, 16, 16384)
        m = _spread(rng, 1, min(65536, MOST_ACTIVATIONS // h // (2 if dtype == "fp32" else 1)))
        return dict(op=op, m=m, h=h, dtype=dtype, params=rng.choice([dtype, "fp32"]), affine=rng.random() < 0.85,
                    strided=rng.random() < 0.25, train=train)
    h = _width(rng, 16, 8192)
    part = 2 if dtype == "fp32" else 1
    v = _spread(rng, 2, min(262144, MOST_TABLE // h // part))
    n = _spread(rng, 1, min(65536, MOST_LOOKED_UP // h // part))
    return dict(op=op, n=n, v=v, h=h, dtype=dtype, padding=rng.random() < 0.4, train=train)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[c["dtype"]]
    s = {"case": c}
    if c["op"] == "route":
        m, e = c["m"], c["e"]
        # a router whose experts are not equally popular
        s["z"] = (1.5 * _normal(g, m, e) + 0.5 * _normal(g, e)).to(dtype)
        s["mask"] = None
        if c["mask"]:  # the tokens behind each sequence's end, about one in five
            s["mask"] = torch.rand(m, generator=g, device="cuda") < 0.8
        if c["train"]:
            s["z"].requires_grad_()
            s["grads"] = (_normal(g, m, c["k"]), torch.tensor(BALANCE, device="cuda"), torch.tensor(Z_LOSS, device="cuda"))
    elif c["op"] == "norm":
        m, h = c["m"], c["h"]
        wide = h + 24 if c["strided"] else h
        # hidden states: an offset per row, a few large channels
        x = _normal(g, m, wide) * (1 + 7 * (torch.rand(wide, generator=g, device="cuda") < 0.01)) + 0.5 * _normal(g, m, 1)
        s["x"] = x.to(dtype)[:, :h]
        params = DTYPES[c["params"]]
        s["w"] = (1 + 0.2 * _normal(g, h)).to(params) if c["affine"] else None
        s["b"] = (0.2 * _normal(g, h)).to(params) if c["affine"] else None
        if c["train"]:
            s["leaves"] = [t.requires_grad_() for t in (s["x"].detach(), s["w"], s["b"]) if t is not None]
            s["x"] = s["leaves"][0]
            s["grad"] = _normal(g, m, h).to(dtype)
    else:
        n, v, h = c["n"], c["v"], c["h"]
        s["table"] = (_normal(g, v, h) / 40).to(dtype)
        # words by their rank in a text: a few of them are most of it
        u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
        rank = (torch.exp(u * math.log(v + 1.0)) - 1).long().clamp(0, v - 1)
        ids = rank * 7919 % v  # frequent rows do not lie together
        if c["padding"]:
            ids = torch.where(torch.rand(n, generator=g, device="cuda") < 0.15, -torch.ones_like(ids), ids)
        s["ids"] = ids.to(torch.int32)
        s["scale"] = math.sqrt(h)
        if c["train"]:
            s["table"].requires_grad_()
            s["grad"] = _normal(g, n, h).to(dtype)
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _plain_route(s):
    c, z = s["case"], s["z"].detach().float()
    m, e, k = c["m"], c["e"], c["k"]
    here = s["mask"] if s["mask"] is not None else torch.ones(m, dtype=torch.bool, device=z.device)
    n = here.sum().clamp(min=1).float()
    top = z.amax(-1, keepdim=True)
    ex = torch.exp(z - top)
    total = ex.sum(-1, keepdim=True)
    p = torch.where(here[:, None], ex / total, torch.zeros_like(ex))
    lse = torch.where(here, (top + torch.log(total))[:, 0], torch.zeros_like(top[:, 0]))
    _, ids = torch.sort(z, dim=-1, descending=True, stable=True)
    ids = ids[:, :k]
    picked = p.gather(1, ids)
    most = picked.sum(-1, keepdim=True)
    w = torch.where(here[:, None], picked / most, torch.zeros_like(picked)) if c["renorm"] else picked
    chosen = torch.zeros(m, e, device=z.device).scatter_(1, ids, 1.0) * here[:, None].float()
    counts = chosen.sum(0)
    load = p.double().sum(0).float()
    balance = (counts / n * load / n).sum() * (e / k)
    z_loss = (lse.double() ** 2).sum().float() / n
    out = (w, torch.where(here[:, None], ids, -torch.ones_like(ids)).to(torch.int32), counts.to(torch.int32), balance, z_loss)
    if not c["train"]:
        return out
    gw, gb, gz = s["grads"]
    pull = (gb * (e / k) / n * counts / n)[None, :].expand(m, e)
    if c["renorm"]:
        direct = torch.zeros_like(p).scatter_(1, ids, w * (gw - (gw * w).sum(-1, keepdim=True)))
    else:
        pull = pull.scatter_add(1, ids, gw)
        direct = torch.zeros_like(p)
    grad = p * (pull - (pull * p).sum(-1, keepdim=True)) + direct + (2 * gz / n) * lse[:, None] * p
    return (*out, torch.where(here[:, None], grad, torch.zeros_like(grad)).to(s["z"].dtype))


def _plain_norm(s):
    c, x = s["case"], s["x"].detach().float()
    mean = x.mean(-1, keepdim=True)
    centred = x - mean
    rstd = 1 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    xhat = centred * rstd
    w = None if s["w"] is None else s["w"].detach().float()
    y = xhat if w is None else xhat * w + s["b"].detach().float()
    y = y.to(s["x"].dtype)
    if not c["train"]:
        return y
    g = s["grad"].float()
    wg = g if w is None else g * w
    dx = rstd * (wg - wg.mean(-1, keepdim=True) - xhat * (wg * xhat).mean(-1, keepdim=True))
    grads = [dx.to(s["x"].dtype)]
    if w is not None:
        grads += [(g * xhat).sum(0).to(s["w"].dtype), g.sum(0).to(s["b"].dtype)]
    return (y, *grads)


def _plain_embed(s):
    c, table, ids = s["case"], s["table"].detach(), s["ids"].long()
    v, h = table.shape
    here = (ids >= 0) & (ids < v)
    at = torch.where(here, ids, torch.zeros_like(ids))
    rows = table[at].float() * s["scale"]
    out = torch.where(here[:, None], rows, torch.zeros_like(rows)).to(table.dtype)
    if not c["train"]:
        return out
    wide = torch.float64 if c["n"] > 16 * v else torch.float32  # long sums
    total = torch.zeros(v + 1, h, dtype=wide, device=table.device)
    total.index_add_(0, torch.where(here, ids, torch.full_like(ids, v)), s["grad"].to(wide))
    return out, (total[:v] * s["scale"]).to(table.dtype)


# ---------------------------------------------------------------------------
# the package's calls
# ---------------------------------------------------------------------------
def _own_route(s):
    import mtp_b200

    c = s["case"]
    r = mtp_b200.route_tokens(s["z"], c["k"], c["renorm"], token_mask=s["mask"])
    if not c["train"]:
        return tuple(r)
    (grad,) = torch.autograd.grad((r.weights, r.balance_loss, r.z_loss), s["z"], s["grads"])
    return r.weights.detach(), r.ids, r.counts, r.balance_loss.detach(), r.z_loss.detach(), grad


def _own_norm(s):
    import mtp_b200

    y = mtp_b200.layer_norm(s["x"], s["w"], s["b"], EPS)
    if not s["case"]["train"]:
        return y
    return (y.detach(), *torch.autograd.grad(y, s["leaves"], s["grad"]))


def _own_embed(s):
    import mtp_b200

    out = mtp_b200.embed_tokens(s["ids"], s["table"], s["scale"])
    if not s["case"]["train"]:
        return out
    return (out.detach(), *torch.autograd.grad(out, s["table"], s["grad"]))


PLAIN = {"route": _plain_route, "norm": _plain_norm, "embed": _plain_embed}
OWN = {"route": _own_route, "norm": _own_norm, "embed": _own_embed}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------
def work(case):
    c, size = case, BYTES[case["dtype"]]
    if c["op"] == "route":
        logits = c["m"] * c["e"]
        b = logits * size + c["m"] * c["k"] * 8 + c["e"] * 4 + 8 + (c["m"] if c["mask"] else 0)
        f = 6 * logits
        if c["train"]:
            b, f = b + logits * size + c["m"] * c["k"] * 4, f + 8 * logits
        return {"bytes": b, "flops": f}
    if c["op"] == "norm":
        rows, params = c["m"] * c["h"], 2 * c["h"] * BYTES[c["params"]] if c["affine"] else 0
        b, f = 2 * rows * size + params, 8 * rows
        if c["train"]:
            b, f = b + 2 * rows * size + params, f + 14 * rows
        return {"bytes": b, "flops": f}
    rows = c["n"] * c["h"]
    read = min(c["n"], _distinct(c["v"], c["n"])) * c["h"] * size
    b, f = read + rows * size + 4 * c["n"], rows
    if c["train"]:
        b, f = b + rows * size + c["v"] * c["h"] * size, f + 2 * rows
    return {"bytes": b, "flops": f}


def _distinct(v, n):
    """Rows that n tokens reach, on average: rank r comes with probability log((r + 1) / r) / log(v + 1)."""
    rank = torch.arange(1, v + 1, dtype=torch.float64)
    return int((1 - (1 - torch.log1p(1 / rank) / math.log(v + 1)) ** n).sum())


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "route":
        with torch.enable_grad():
            return _exact_route(s)
    if c["op"] == "norm":
        with torch.enable_grad():
            return _exact_norm(s)
    with torch.no_grad():
        table, ids = s["table"].double(), s["ids"].long()
        inside = ((ids >= 0) & (ids < c["v"])).nonzero()[:, 0]
        out = torch.zeros(c["n"], c["h"], dtype=torch.float64, device="cuda")
        out[inside] = s["scale"] * table[ids[inside]]
        if not c["train"]:
            return out
        del table
        total = torch.zeros(c["v"], c["h"], dtype=torch.float64, device="cuda")
        total.index_put_((ids[inside],), s["grad"][inside].double(), accumulate=True)
        return out, total * s["scale"]


def _exact_route(s):
    """By differentiation of the definition."""
    c = s["case"]
    z = s["z"].detach().double().requires_grad_()
    rows = z if s["mask"] is None else z[s["mask"]]
    n = rows.shape[0]
    p = torch.softmax(rows, -1)
    # the k largest, lowest id first where equal: by a key that has no ties
    key = s["z"].detach().double() if s["mask"] is None else s["z"].detach().double()[s["mask"]]
    ids = torch.argsort(-key, dim=-1, stable=True)[:, : c["k"]]
    w = torch.gather(p, 1, ids)
    if c["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    counts = torch.bincount(ids.flatten(), minlength=c["e"]).double()
    balance = (c["e"] / c["k"] / max(n, 1) ** 2) * (counts @ p.sum(0))
    z_loss = torch.logsumexp(rows, -1).square().sum() / max(n, 1)
    full = w if s["mask"] is None else torch.zeros(c["m"], c["k"], dtype=torch.float64, device="cuda").index_put((s["mask"].nonzero()[:, 0],), w)
    out = (full.detach(), None, None, balance.detach(), z_loss.detach())
    if not c["train"]:
        return out
    gw, gb, gz = (g.double() for g in s["grads"])
    loss = (full * gw).sum() + gb * balance + gz * z_loss
    return (*out, *torch.autograd.grad(loss, z))


def _exact_norm(s):
    """By differentiation of the definition."""
    leaves = [None if t is None else t.detach().double().requires_grad_() for t in (s["x"], s["w"], s["b"])]
    x, w, b = leaves
    y = (x - x.mean(-1, keepdim=True)) / (x.var(-1, unbiased=False, keepdim=True) + EPS).sqrt()
    if w is not None:
        y = y * w + b
    if not s["case"]["train"]:
        return y.detach()
    return (y.detach(), *torch.autograd.grad(y, [t for t in leaves if t is not None], s["grad"].double()))

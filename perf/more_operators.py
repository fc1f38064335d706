"""Performance cases of the operators at the two ends of a decoder's training step.

A case is one call, or for training one forward and backward step, of

* ``embed``       scaled rows of an embedding table (``ops.embedding``);
* ``embed_grad``  the table's gradient (``ops.embeddingGrad``);
* ``norm``        layer norm (``ops.layerNorm``);
* ``norm_grad``   the same with its gradients (``ops.layerNormGrad``);
* ``loss``        softmax cross entropy of a linear head (``ops.linearCrossEntropy``);
* ``loss_grad``   the same with its gradients (``ops.linearCrossEntropyGrad``).

``run`` makes these calls where ``own`` is true and computes the same in elementary torch
operations, in float32, where it is false; ``exact`` computes them in float64 from the
definitions.  Sizes follow from the case alone, all values, ids and targets from the seed.
"""
from __future__ import annotations

import math

import torch

own = False

_TORCH = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


def listed():
    return [
        # the tokens of one short question: latency counts
        {"name": "embed_short", "kind": "embed", "dtype": "float16", "tokens": 37,
         "vocab": 32000, "width": 1024, "scaled": True},
        # a batch of documents packed to 16384 tokens
        {"name": "embed_batch", "kind": "embed", "dtype": "bfloat16", "tokens": 16384,
         "vocab": 128256, "width": 4096, "scaled": True},
        # the gradient of a small float32 table: latency counts
        {"name": "embed_grad_short", "kind": "embed_grad", "dtype": "float32", "tokens": 300,
         "vocab": 1001, "width": 250, "scaled": False},
        # the gradient of a large table: a few tokens often, most never
        {"name": "embed_grad_batch", "kind": "embed_grad", "dtype": "bfloat16", "tokens": 16384,
         "vocab": 128256, "width": 4096, "scaled": True},
        # the norm of a few chats' next tokens: latency counts
        {"name": "norm_short", "kind": "norm", "dtype": "bfloat16", "rows": 16, "width": 4096,
         "params": "float32"},
        # a training step's norm over 8192 tokens
        {"name": "norm_train", "kind": "norm_grad", "dtype": "bfloat16", "rows": 8192,
         "width": 4096, "params": "float32"},
        # a small float32 model's, rows of an odd width
        {"name": "norm_odd", "kind": "norm_grad", "dtype": "float32", "rows": 2000,
         "width": 1001, "params": "float32"},
        # few rows that are very wide
        {"name": "norm_wide", "kind": "norm_grad", "dtype": "float16", "rows": 300,
         "width": 20000, "params": "float16"},
        # a small model's step on a few sentences: latency counts
        {"name": "loss_short", "kind": "loss_grad", "dtype": "float16", "tokens": 100,
         "hidden": 256, "vocab": 1000, "tied": False},
        # the evaluation of a tied model of an odd vocabulary
        {"name": "loss_eval", "kind": "loss", "dtype": "bfloat16", "tokens": 2000,
         "hidden": 1024, "vocab": 50257, "tied": True},
        # a training step of a tied model
        {"name": "loss_tied", "kind": "loss_grad", "dtype": "float16", "tokens": 4000,
         "hidden": 2048, "vocab": 32003, "tied": True},
        # a training step of a large vocabulary's own head
        {"name": "loss_train", "kind": "loss_grad", "dtype": "bfloat16", "tokens": 8192,
         "hidden": 4096, "vocab": 128256, "tied": False},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["embed", "embed_grad", "norm", "norm_grad", "loss", "loss_grad",
                       "loss_grad"])
    c = {"kind": kind}
    if kind in ("embed", "embed_grad"):
        c["dtype"] = rng.choice(["bfloat16", "float16", "float32"])
        c["tokens"], c["vocab"] = _log(rng, 1, 16384), _log(rng, 2, 128256)
        c["width"] = rng.choice([_log(rng, 1, 4000), 64 * _log(rng, 1, 64)])
        if c["dtype"] == "float32":
            c["vocab"] = min(c["vocab"], 64000)
        c["scaled"] = rng.random() < 0.5
    elif kind in ("norm", "norm_grad"):
        c["dtype"] = rng.choice(["bfloat16", "float16", "float32"])
        c["width"] = rng.choice([_log(rng, 1, 20000), 64 * _log(rng, 1, 256)])
        c["rows"] = _log(rng, 1, max(1, min(16384, 8192 * 4096 // c["width"])))
        c["params"] = rng.choice([c["dtype"], "float32"])
    else:
        c["dtype"] = rng.choice(["bfloat16", "float16"])
        c["tokens"] = _log(rng, 1, 8192)
        c["hidden"] = rng.choice([_log(rng, 1, 4000), 64 * _log(rng, 1, 64)])
        c["vocab"] = rng.choice([_log(rng, 2, 128000), 8 * _log(rng, 1, 16000)])
        c["tied"] = rng.random() < 0.5
    return c


# ---- inputs ------------------------------------------------------------------------------

def _normal(gen, shape, dtype, std=1.0, mean=0.0):
    return torch.empty(shape, dtype=_TORCH[dtype], device="cuda").normal_(mean, std,
                                                                          generator=gen)


def _ids(gen, n, vocab):
    """Ids as text has them: id v about as often as 1 / (v + 1), in a mixed order of ids; one
    in twenty belongs to padding and is -1."""
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    v = (torch.exp(u * math.log(vocab + 1.0)) - 1.0).long().clamp(0, vocab - 1)
    v = torch.randperm(vocab, generator=gen, device="cuda")[v]
    pad = torch.rand(n, generator=gen, device="cuda") < 0.05
    return torch.where(pad, -1, v).to(torch.int32)


def _make(c, seed):
    """The case's inputs as torch tensors, and the numbers that a program knows beside them."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind = c["kind"]
    if kind in ("embed", "embed_grad"):
        n, vocab, width = c["tokens"], c["vocab"], c["width"]
        known = {"vocab": vocab, "scale": math.sqrt(width) if c["scaled"] else 1.0}
        x = {"ids": _ids(gen, n, vocab)}
        if kind == "embed":
            x["weight"] = _normal(gen, (vocab, width), c["dtype"], 1.0 / math.sqrt(width))
        else:
            x["grad"] = _normal(gen, (n, width), c["dtype"], 0.01)
        return x, known
    if kind in ("norm", "norm_grad"):
        n, width = c["rows"], c["width"]
        x = {"x": _normal(gen, (n, width), c["dtype"], 1.5, 0.25),
             "gamma": _normal(gen, (width,), c["params"], 0.1, 1.0),
             "beta": _normal(gen, (width,), c["params"], 0.1)}
        if kind == "norm_grad":
            x["grad"] = _normal(gen, (n, width), c["dtype"], 0.01)
        return x, {"eps": 1e-5}
    n, hidden, vocab = c["tokens"], c["hidden"], c["vocab"]
    shape = (vocab, hidden) if c["tied"] else (hidden, vocab)
    x = {"x": _normal(gen, (n, hidden), c["dtype"]),
         "weight": _normal(gen, shape, c["dtype"], 2.0 / math.sqrt(hidden)),
         "targets": _ids(gen, n, vocab)}
    if kind == "loss_grad":  # the mean over weighted tokens; float16 training scales its loss
        w = 0.5 + torch.rand(n, generator=gen, device="cuda")
        x["grad"] = w / n * (4096.0 if c["dtype"] == "float16" else 1.0)
    return x, {"tied": c["tied"]}


class _Memory:
    """A framework tensor's device memory under the array interface that torch reads."""

    __slots__ = ("__cuda_array_interface__", "tensor")


def _view(t):
    """A framework tensor's memory as a torch tensor (no copy; it keeps `t` alive)."""
    from rew_amd import eager as E
    m = _Memory()
    m.tensor = t
    m.__cuda_array_interface__ = {"shape": t.shape, "typestr": "<f4" if t.dtype == E.float32
                                  else "<i4" if t.dtype == E.int32 else "<i2", "version": 2,
                                  "data": (E.devicePtr(t), False)}
    v = torch.as_tensor(m, device="cuda")
    return v if v.dtype != torch.int16 else v.view(
        torch.bfloat16 if t.dtype == E.bfloat16 else torch.float16)


def _tensor(x):
    """A framework tensor with the values of a torch tensor."""
    from rew_amd import eager as E
    t = E.empty({torch.bfloat16: E.DType.BFLOAT16, torch.float16: E.DType.FLOAT16,
                 torch.float32: E.DType.FLOAT32, torch.int32: E.DType.INT32}[x.dtype],
                tuple(x.shape))
    _view(t).copy_(x)
    return t


def prepare(case, seed):
    x, known = _make(case, seed)
    if own:  # a program of the framework has the same values in the framework's tensors
        from rew_amd import eager as E
        E.installEagerBackend()
        x = {k: _tensor(v) for k, v in x.items()}
        torch.cuda.synchronize()
    return {"kind": case["kind"], "x": x, "known": known}


# ---- one pass ------------------------------------------------------------------------------

def run(state):
    kind, x, known = state["kind"], state["x"], state["known"]
    if own:
        return _calls(kind, x, known)
    return _PLAIN[kind](x, known)


def _calls(kind, x, known):
    from rew_amd import ops as O
    if kind == "embed":
        return _view(O.embedding(x["weight"], x["ids"], scale=known["scale"]))
    if kind == "embed_grad":
        return _view(O.embeddingGrad(x["ids"], x["grad"], known["vocab"],
                                     scale=known["scale"]))
    if kind == "norm":
        return _view(O.layerNorm(x["x"], x["gamma"], x["beta"], eps=known["eps"]))
    if kind == "norm_grad":
        y, stats = O.layerNorm(x["x"], x["gamma"], x["beta"], eps=known["eps"], withStats=True)
        got = O.layerNormGrad(x["x"], x["gamma"], stats, x["grad"])
        return [_view(t) for t in (y, *got)]
    if kind == "loss":
        return _view(O.linearCrossEntropy(x["x"], x["weight"], x["targets"],
                                          tied=known["tied"]))
    loss, lse = O.linearCrossEntropy(x["x"], x["weight"], x["targets"], tied=known["tied"],
                                     withLse=True)
    got = O.linearCrossEntropyGrad(x["x"], x["weight"], x["targets"], lse, x["grad"],
                                   tied=known["tied"])
    return [_view(t) for t in (loss, *got)]


def _plain_embed(x, known):
    w, ids = x["weight"], x["ids"].long()
    there = (ids >= 0) & (ids < w.shape[0])
    rows = w[ids.clamp(0, w.shape[0] - 1)].float() * (there[:, None] * known["scale"])
    return rows.to(w.dtype)


def _plain_embed_grad(x, known):
    g, ids, vocab = x["grad"], x["ids"].long(), known["vocab"]
    there = (ids >= 0) & (ids < vocab)
    # ids outside the table go to a row behind it
    out = torch.zeros((vocab + 1, g.shape[1]), dtype=torch.float32, device=g.device)
    out.index_add_(0, torch.where(there, ids, vocab), g.float())
    return (out[:vocab] * known["scale"]).to(g.dtype)


def _plain_norm_parts(x, known):
    v = x["x"].float()
    mean = v.mean(1, keepdim=True)
    c = v - mean
    rstd = torch.rsqrt((c * c).mean(1, keepdim=True) + known["eps"])
    return c * rstd, rstd


def _plain_norm(x, known):
    h, _ = _plain_norm_parts(x, known)
    return (h * x["gamma"].float() + x["beta"].float()).to(x["x"].dtype)


def _plain_norm_grad(x, known):
    h, rstd = _plain_norm_parts(x, known)
    gamma, dy = x["gamma"].float(), x["grad"].float()
    y = h * gamma + x["beta"].float()
    w = dy * gamma
    dx = rstd * (w - w.mean(1, keepdim=True) - h * (w * h).mean(1, keepdim=True))
    return [y.to(x["x"].dtype), dx.to(x["x"].dtype), (dy * h).sum(0).to(x["gamma"].dtype),
            dy.sum(0).to(x["gamma"].dtype)]


def _plain_loss_parts(x, known):
    """The float32 logits less their largest, the sums of their exponentials, the loss."""
    w, t = x["weight"].float(), x["targets"].long()
    z = x["x"].float() @ (w.t() if known["tied"] else w)
    there = (t >= 0) & (t < z.shape[1])
    t = t.clamp(0, z.shape[1] - 1)
    z -= z.amax(1, keepdim=True)
    at = z.gather(1, t[:, None])[:, 0]
    e = z.exp_()
    total = e.sum(1)
    return w, e, total, there, t, torch.where(there, torch.log(total) - at, 0.0)


def _plain_loss(x, known):
    return _plain_loss_parts(x, known)[-1]


def _plain_loss_grad(x, known):
    w, e, total, there, t, loss = _plain_loss_parts(x, known)
    g = x["grad"] * there
    dz = e.mul_((g / total)[:, None])
    dz.scatter_add_(1, t[:, None], -g[:, None])
    v, dt = x["x"].float(), x["x"].dtype
    if known["tied"]:
        return [loss, (dz @ w).to(dt), (dz.t() @ v).to(dt)]
    return [loss, (dz @ w.t()).to(dt), (v.t() @ dz).to(dt)]


_PLAIN = {"embed": _plain_embed, "embed_grad": _plain_embed_grad, "norm": _plain_norm,
          "norm_grad": _plain_norm_grad, "loss": _plain_loss, "loss_grad": _plain_loss_grad}


# ---- what a pass has to move and compute ---------------------------------------------------

_BYTES = {"bfloat16": 2, "float16": 2, "float32": 4}


def work(case):
    kind, size = case["kind"], _BYTES[case["dtype"]]
    if kind == "embed":  # each used row of the table is read once
        n, vocab = case["tokens"], case["vocab"]
        used = int(min(n, sum(1 - (1 - 1 / ((v + 1) * math.log(vocab + 1))) ** (0.95 * n)
                              for v in range(vocab))))
        return {"bytes": (n + used) * case["width"] * size + 4 * n, "flops": 0}
    if kind == "embed_grad":
        n = case["tokens"]
        return {"bytes": (n + case["vocab"]) * case["width"] * size + 4 * n,
                "flops": n * case["width"]}
    if kind in ("norm", "norm_grad"):
        n, params = case["rows"] * case["width"], _BYTES[case["params"]] * case["width"]
        if kind == "norm":
            return {"bytes": 2 * n * size + 2 * params, "flops": 8 * n}
        # x, gradOut, y and gradX; gamma, beta and their gradients
        return {"bytes": 4 * n * size + 4 * params, "flops": 20 * n}
    t, h, v = case["tokens"], case["hidden"], case["vocab"]
    if kind == "loss":
        return {"bytes": size * (t * h + h * v) + 8 * t, "flops": 2 * t * h * v}
    # the logits, and their gradient times x and the weight
    return {"bytes": 2 * size * (t * h + h * v) + 12 * t, "flops": 6 * t * h * v}


# ---- the definitions in 64 bits --------------------------------------------------------------

def _exact_rows(x, known, kind):
    """Layer norm and its gradients, from the moments E[x], E[x^2] about the row's first
    value and the derivative of each."""
    v = x["x"].double()
    first = v[:, :1].clone()
    d = v - first
    m1, m2 = d.mean(1, keepdim=True), (d * d).mean(1, keepdim=True)
    var = (m2 - m1 * m1).clamp(min=0.0)
    sd = torch.sqrt(var + known["eps"])
    gamma, beta = x["gamma"].double(), x["beta"].double()
    y = (d - m1) / sd * gamma + beta
    if kind == "norm":
        return y
    dy = x["grad"].double()
    u = dy * gamma
    # y depends on x_j directly, through m1 and through var
    d_var = (u * (d - m1)).sum(1, keepdim=True) * (-0.5) / sd ** 3
    d_m1 = -u.sum(1, keepdim=True) / sd
    n = v.shape[1]
    dx = u / sd + d_m1 / n + d_var * 2.0 * (d - m1) / n
    return [y, dx, torch.einsum("rc,rc->c", dy, (d - m1) / sd), torch.ones(
        v.shape[0], dtype=torch.float64, device=v.device) @ dy]


def _exact_loss(x, known, kind):
    """Token block by token block, p from logsumexp."""
    w = x["weight"].double()
    w = w.t() if known["tied"] else w                      # [hidden, vocab]
    hidden, vocab = w.shape
    n = x["x"].shape[0]
    loss = torch.zeros(n, dtype=torch.float64, device=w.device)
    dx = torch.zeros((n, hidden), dtype=torch.float64, device=w.device)
    dw = torch.zeros((hidden, vocab), dtype=torch.float64, device=w.device) \
        if kind == "loss_grad" else None
    step = max(1, min(n, 2 ** 28 // vocab))
    for at in range(0, n, step):
        rows = slice(at, min(n, at + step))
        v, t = x["x"][rows].double(), x["targets"][rows].long()
        live = ((t >= 0) & (t < vocab)).nonzero()[:, 0]
        z = v[live] @ w
        lse = torch.logsumexp(z, 1)
        hit = (torch.arange(len(live), device=w.device), t[live])
        part = torch.zeros(len(t), dtype=torch.float64, device=w.device)
        part[live] = lse - z[hit]
        loss[rows] = part
        if kind == "loss_grad":
            p = torch.exp(z - lse[:, None])
            p[hit] -= 1.0
            p *= x["grad"][rows][live].double()[:, None]
            dx[at + live] = p @ w.t()
            dw += v[live].t() @ p
    if kind == "loss":
        return loss
    return [loss, dx, dw.t().contiguous() if known["tied"] else dw]


def exact(case, seed):
    kind = case["kind"]
    x, known = _make(case, seed)
    if kind in ("norm", "norm_grad"):
        return _exact_rows(x, known, kind)
    if kind in ("loss", "loss_grad"):
        return _exact_loss(x, known, kind)
    ids = x["ids"].long()
    live = ((ids >= 0) & (ids < known["vocab"])).nonzero()[:, 0]
    if kind == "embed":
        out = torch.zeros((len(ids), x["weight"].shape[1]), dtype=torch.float64, device="cuda")
        out[live] = x["weight"].double()[ids[live]] * known["scale"]
        return out
    # the rows in the order of their ids, summed run by run
    order = live[torch.argsort(ids[live], stable=True)]
    runs, counts = torch.unique_consecutive(ids[order], return_counts=True)
    sums = torch.segment_reduce(x["grad"].double()[order], "sum", lengths=counts, axis=0)
    out = torch.zeros((known["vocab"], x["grad"].shape[1]), dtype=torch.float64, device="cuda")
    out[runs] = sums * known["scale"]
    return out

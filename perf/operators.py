"""What is measured of the operators around the circuit layers: layer norm with its gradients, the clipping of gradients by their
global norm, and sampling of symbols from log-probabilities.

A network that predicts a circuit's weights normalises its activations (`layer_norm`, `layer_norm_backward`), its training step
clips the gradients of all layers by their common norm (`clip_grad_norm_`), and the log-probabilities that the circuit gives
the symbols are sampled from (`sample`).  A case is one call on tensors that are resident on the GPU; a training step of the
layer norm is its two calls.
"""

import math
import random

import torch

own = False

NEG_INF = float("-inf")
_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_SIGMA = 0.02  # standard deviation of a gradient's elements


def listed():
    return [
        # One small batch of hidden activations, odd in both sizes: the latency of a call.
        {"name": "norm 9x1000 f32", "op": "norm", "step": False, "rows": 9, "width": 1000, "type": "float32"},
        # The forward pass alone, as in evaluation, over a large batch.
        {"name": "norm 16384x2048 bf16", "op": "norm", "step": False, "rows": 16384, "width": 2048, "type": "bfloat16"},
        # Training in 32 bits, sizes that no vector load divides.
        {"name": "norm step 5003x1537 f32", "op": "norm", "step": True, "rows": 5003, "width": 1537, "type": "float32"},
        # Training of wide layers over a large batch: the longest step.
        {"name": "norm step 16384x8192 bf16", "op": "norm", "step": True, "rows": 16384, "width": 8192, "type": "bfloat16"},
        # The few small tensors of one circuit's layers: launches count.
        {"name": "clip 12 small f32", "op": "clip", "tensors": 12, "numbers": 40000, "type": "float32", "norm": 2.0, "above": True},
        # The layers of a medium model in 32 bits, sizes spread over three decades, the norm above the limit.
        {"name": "clip 60 f32", "op": "clip", "tensors": 60, "numbers": 30_000_000, "type": "float32", "norm": 2.0, "above": True},
        # The same model later in training: the norm is within the limit and nothing has to change.
        {"name": "clip 60 f32 within", "op": "clip", "tensors": 60, "numbers": 30_000_000, "type": "float32", "norm": 2.0, "above": False},
        # A large model with 16-bit weights and a few 32-bit ones.
        {"name": "clip 40 mixed", "op": "clip", "tensors": 40, "numbers": 700_000_000, "type": "mixed", "norm": 2.0, "above": True},
        # One answer of an interactive program.
        {"name": "sample 1x32768 f32", "op": "sample", "rows": 1, "symbols": 32768, "type": "float32", "filters": "k50 p0.9", "per_row": False},
        # A batch of requests, each with parameters of its own, over an odd number of symbols.
        {"name": "sample 64x50021 bf16", "op": "sample", "rows": 64, "symbols": 50021, "type": "bfloat16", "filters": "k p m", "per_row": True},
        # Many samples of the whole distribution: nothing is filtered.
        {"name": "sample 200x10007 f32", "op": "sample", "rows": 200, "symbols": 10007, "type": "float32", "filters": "", "per_row": False},
        # A large batch over many symbols, by mass alone: the largest call.
        {"name": "sample 256x131072 f32", "op": "sample", "rows": 256, "symbols": 131072, "type": "float32", "filters": "p0.95", "per_row": False},
    ]  # fmt: skip


def _between(rng, low, high):
    """A whole number of the range, spread over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["norm", "clip", "sample"])
    if op == "norm":
        while True:
            rows, width = _between(rng, 1, 40000), _between(rng, 64, 16384)
            width = max(64, width // 64 * 64) if rng.random() < 0.5 else width
            if rows * width <= 16384 * 8192:
                break
        kind = rng.choice(list(_TYPES))
        return {"op": op, "step": rng.random() < 0.6, "rows": rows // (2 if kind == "float32" and rows > 1 else 1), "width": width, "type": kind}
    if op == "clip":
        tensors = _between(rng, 1, 60)
        kind = rng.choice(["float32", "bfloat16", "mixed"])
        numbers = _between(rng, 64 * tensors, 300_000_000)
        return {"op": op, "tensors": tensors, "numbers": numbers, "type": kind, "norm": rng.choice([2.0, 2.0, math.inf]), "above": rng.random() < 0.7}
    while True:
        rows, symbols = _between(rng, 1, 256), _between(rng, 500, 200_000)
        if rows * symbols <= 256 * 131072:
            break
    filters = rng.choice(["", "k50", "p0.9", "m0.05", "k200 p0.95", "k50 p0.9 m0.02", "k p m"])
    return {"op": op, "rows": rows, "symbols": symbols, "type": rng.choice(list(_TYPES)), "filters": filters, "per_row": filters == "k p m"}


# ----------------------------------------------------------------------------- inputs


def _sizes(case):
    """Numbers of elements of the tensors whose gradients are clipped: spread over three decades, `numbers` in all."""
    rng = random.Random(case["tensors"] * 1_000_003 + case["numbers"])
    share = [10.0 ** rng.uniform(-3.0, 0.0) for _ in range(case["tensors"])]
    return [max(1, int(case["numbers"] * s / sum(share))) for s in share]


def _kinds(case):
    """Element types of those tensors: "mixed" keeps the smaller half in 32 bits and has the others in 16."""
    sizes = _sizes(case)
    if case["type"] != "mixed":
        return [_TYPES[case["type"]]] * len(sizes)
    middle = sorted(sizes)[len(sizes) // 2]
    return [torch.float32 if n < middle else torch.bfloat16 for n in sizes]


def _filters(case):
    """ "k50 p0.9" as {"k": "50", "p": "0.9"}: top-k, top-p and min-p (m) by their first letters."""
    return {f[0]: f[1:] for f in case["filters"].split()}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.rand(*s, generator=g, device="cuda")  # noqa: E731
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    if case["op"] == "norm":
        kind, rows, width = _TYPES[case["type"]], case["rows"], case["width"]
        # activations: features at levels and scales of their own, a few of them large
        level = 0.3 * randn(width)
        scale = torch.exp(0.4 * randn(width)) * torch.where(rand(width) < 0.01, 8.0, 1.0)
        x = (randn(rows, width) * scale + level).to(kind)
        state = {"op": "norm", "step": case["step"], "x": x, "weight": (1.0 + 0.1 * randn(width)).to(kind), "bias": (0.1 * randn(width)).to(kind)}
        if case["step"]:
            state["dy"] = (0.05 * randn(rows, width)).to(kind)
        return state
    if case["op"] == "clip":
        grads = [(_SIGMA * randn(n)).to(kind) for n, kind in zip(_sizes(case), _kinds(case))]
        total = sum(_sizes(case))
        norm = _SIGMA * math.sqrt(total) if case["norm"] == 2.0 else _SIGMA * math.sqrt(2.0 * math.log(total + 1.0))
        # (another seed is another limit too: a program's schedule moves it)
        limit = norm * (0.5 if case["above"] else 4.0) * (1.0 + 1e-3 * (seed % 97))
        # A pass clips in place, so that the next one on the same tensors would find them within the limit.  New gradients would
        # not be: the limit falls by a little from pass to pass, so that every pass finds a norm above it.
        return {"op": "clip", "grads": grads, "limit": limit, "falls": 0.9999 if case["above"] else 1.0, "norm": case["norm"]}
    kind, rows, symbols = _TYPES[case["type"]], case["rows"], case["symbols"]
    # log-probabilities as a circuit gives them, some symbols impossible
    logits = torch.log_softmax(3.0 * randn(rows, symbols), dim=-1)
    logits = logits.masked_fill_(rand(rows, symbols) < 0.01, NEG_INF).to(kind)
    noise = torch.empty(rows, symbols, device="cuda").exponential_(generator=g)
    given = _filters(case)
    state = {"op": "sample", "logits": logits, "noise": noise, "temperature": 0.8, "top_k": None, "top_p": None, "min_p": None}
    if case["per_row"]:
        state["temperature"] = 0.5 + 0.8 * rand(rows)
        state["top_k"] = torch.where(rand(rows) < 0.3, symbols, (10 + 200 * rand(rows)).long()).to(torch.int32)
        state["top_p"] = torch.where(rand(rows) < 0.3, torch.ones(rows, device="cuda"), 0.7 + 0.3 * rand(rows))
        state["min_p"] = torch.where(rand(rows) < 0.5, torch.zeros(rows, device="cuda"), 0.1 * rand(rows))
    else:
        state["top_k"] = int(given["k"]) if "k" in given else None
        state["top_p"] = float(given["p"]) if "p" in given else None
        state["min_p"] = float(given["m"]) if "m" in given else None
    return state


# ----------------------------------------------------------------------------- plain forms


def _plain_norm(x, weight, bias, eps):
    f = x.float()
    mean = f.mean(-1, keepdim=True)
    c = f - mean
    rstd = torch.rsqrt((c * c).mean(-1, keepdim=True) + eps)
    y = (c * rstd) * weight.float() + bias.float()
    return y.to(x.dtype), mean.squeeze(-1), rstd.squeeze(-1)


def _plain_norm_backward(dy, x, mean, rstd, weight):
    d = dy.float()
    h = (x.float() - mean[:, None]) * rstd[:, None]
    g = d * weight.float()
    dx = rstd[:, None] * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    return dx.to(x.dtype), (d * h).sum(0).to(weight.dtype), d.sum(0).to(weight.dtype)


def _plain_clip(grads, limit, norm):
    if norm == 2.0:
        total = torch.stack([g.float().square().sum() for g in grads]).sum().sqrt()
    else:
        total = torch.stack([g.float().abs().max() for g in grads]).max()
    factor = torch.clamp(limit / (total + 1e-6), max=1.0)
    return [g.copy_(g.float() * factor) for g in grads], total


def _column(v):
    return v[:, None] if isinstance(v, torch.Tensor) else v


def _plain_sample(logits, noise, temperature, top_k, top_p, min_p):
    x, order = torch.sort(logits.float() / _column(temperature), dim=-1, descending=True, stable=True)
    p = torch.exp(x - x[:, :1])
    if top_k is not None:
        rank = torch.arange(p.shape[1], device=p.device)
        p = torch.where(rank < _column(top_k), p, 0.0)
    if top_p is not None:
        before = torch.cumsum(p, -1) - p
        share = torch.as_tensor(_column(top_p), device=p.device)
        p = torch.where((before < share * p.sum(-1, keepdim=True)) | (share >= 1.0), p, 0.0)
    if min_p is not None:
        p = torch.where(p >= _column(min_p), p, 0.0)
    best = torch.argmax(p / noise.gather(1, order), dim=-1, keepdim=True)
    return order.gather(1, best).squeeze(-1), torch.log(p.gather(1, best) / p.sum(-1, keepdim=True)).squeeze(-1)


def run(state):
    if own:
        import triturus_b200 as tb
    if state["op"] == "norm":
        x, weight, bias = state["x"], state["weight"], state["bias"]
        if not state["step"]:
            return {"y": tb.layer_norm(x, weight, bias) if own else _plain_norm(x, weight, bias, 1e-5)[0]}
        if own:
            y, mean, rstd = tb.layer_norm(x, weight, bias, return_stats=True)
            dx, dweight, dbias = tb.layer_norm_backward(state["dy"], x, mean, rstd, weight)
        else:
            y, mean, rstd = _plain_norm(x, weight, bias, 1e-5)
            dx, dweight, dbias = _plain_norm_backward(state["dy"], x, mean, rstd, weight)
        return {"y": y, "mean": mean, "rstd": rstd, "dx": dx, "dweight": dweight, "dbias": dbias}
    if state["op"] == "clip":
        limit, grads = state["limit"], state["grads"]
        state["limit"] = limit * state["falls"]
        if own:
            return {"grads": grads, "norm": tb.clip_grad_norm_(grads, limit, norm_type=state["norm"])}
        grads, total = _plain_clip(grads, limit, state["norm"])
        return {"grads": grads, "norm": total}
    names = ("temperature", "top_k", "top_p", "min_p")
    if own:
        token, logprob = tb.sample(state["logits"], state["noise"], **{n: state[n] for n in names}, return_logprob=True)
    else:
        token, logprob = _plain_sample(state["logits"], state["noise"], *(state[n] for n in names))
    return {"token": token, "logprob": logprob}


# ----------------------------------------------------------------------------- definitions in 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "norm":
        x = state["x"].double().requires_grad_(case["step"])
        weight, bias = (state[n].double().requires_grad_(case["step"]) for n in ("weight", "bias"))
        mean = x.sum(-1) / case["width"]
        var = torch.linalg.vecdot(x - mean[:, None], x - mean[:, None]) / case["width"]
        rstd = 1.0 / torch.sqrt(var + 1e-5)
        y = torch.addcmul(bias, (x - mean[:, None]) * rstd[:, None], weight)
        if not case["step"]:
            return {"y": y}
        dx, dweight, dbias = torch.autograd.grad(y, (x, weight, bias), state["dy"].double())
        return {"y": y, "mean": mean, "rstd": rstd, "dx": dx, "dweight": dweight, "dbias": dbias}
    if case["op"] == "clip":
        parts = [torch.linalg.vector_norm(g.double(), ord=case["norm"]) for g in state["grads"]]
        total = torch.linalg.vector_norm(torch.stack(parts), ord=case["norm"])
        factor = min(1.0, state["limit"] / (float(total) + 1e-6))
        return {"grads": [g.double() * factor for g in state["grads"]], "norm": total}
    x = state["logits"].double() / (_column(state["temperature"]) if not case["per_row"] else state["temperature"].double()[:, None])
    # The kept symbols are those above a threshold, and of those at it the first few: how many are kept in all is the least of
    # what the filters allow, and the threshold is the value at that rank.
    down = torch.sort(x, dim=-1).values.flip(-1)
    mass = torch.exp(down - torch.logsumexp(x, -1, keepdim=True))
    kept = torch.full((case["rows"],), case["symbols"], device=x.device)
    if state["top_k"] is not None:
        kept = torch.minimum(kept, torch.as_tensor(state["top_k"], device=x.device).long().expand_as(kept))
    if state["top_p"] is not None:
        share = torch.as_tensor(state["top_p"], device=x.device).double().expand(case["rows"])
        upto = torch.cumsum(mass, -1)
        want = share * upto.gather(1, kept[:, None] - 1).squeeze(-1)
        by_mass = 1 + (upto < want[:, None]).sum(-1)
        kept = torch.where(share < 1.0, torch.minimum(kept, by_mass), kept)
    if state["min_p"] is not None:
        least = torch.as_tensor(state["min_p"], device=x.device).double().expand(case["rows"])
        kept = torch.minimum(kept, (down >= down[:, :1] + torch.log(least)[:, None]).sum(-1))
    at = down.gather(1, kept[:, None] - 1)
    first = torch.cumsum(x == at, -1) <= (kept - (x > at).sum(-1))[:, None]
    x = torch.where((x > at) | ((x == at) & first), x, NEG_INF)
    best = torch.argmax(x - torch.log(state["noise"].double()), dim=-1, keepdim=True)
    return {"token": None, "logprob": (x.gather(1, best) - torch.logsumexp(x, -1, keepdim=True)).squeeze(-1)}


# ----------------------------------------------------------------------------- work


def work(case):
    """Inputs read once, outputs written once.

    Layer norm: some 8 operations per element forwards and 14 backwards.  Clipping: every element is read and, where the norm is
    above the limit, written.  Sampling: the logits are read; of the noise, what belongs to the symbols that the filters
    keep, which is all of it where there are none and next to nothing otherwise; an exponential, a product and some comparisons
    per symbol."""
    if case["op"] == "norm":
        n, e = case["rows"] * case["width"], _TYPES[case["type"]].itemsize
        if not case["step"]:
            return {"bytes": 2 * n * e + 2 * case["width"] * e, "flops": 8 * n}
        return {"bytes": 5 * n * e + 8 * case["rows"] + 4 * case["width"] * e, "flops": 22 * n}
    if case["op"] == "clip":
        sizes = _sizes(case)
        nbytes = sum(n * kind.itemsize for n, kind in zip(sizes, _kinds(case)))
        return {"bytes": (2 if case["above"] else 1) * nbytes, "flops": (3 if case["above"] else 2) * sum(sizes)}
    n = case["rows"] * case["symbols"]
    return {"bytes": n * (_TYPES[case["type"]].itemsize + (0 if case["filters"] else 4)), "flops": 8 * n}

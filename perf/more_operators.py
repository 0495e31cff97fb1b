"""What is measured of the two ends of a model over symbols: the lookup of symbols' embeddings with its gradient, and the cross
entropy of a linear layer over many symbols, taken in pieces of them and with its gradients.

A network that is conditioned on symbols reads their rows of a table (`embedding`, `embedding_backward`); one that predicts symbols
is trained on the cross entropy of x W^T (`linear_cross_entropy`, `linear_cross_entropy_backward`), often with the same table as W.  A case is
one call on tensors that are resident on the GPU; a training step is the two calls of its operator.
"""

import math
import random

import numpy as np
import torch

own = False

IGNORED = -100  # the target of a position without a loss
PADDING = 0  # the symbol that fills up short sequences
_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # The symbols of one short request: the latency of a call.
        {"name": "embed 9x1000 f32", "op": "embed", "step": False, "tokens": 9, "width": 1000, "symbols": 10007, "type": "float32", "scale": 1.0, "padded": False},
        # A batch of prompts, scaled by the root of the width.
        {"name": "embed 16384x2048 bf16", "op": "embed", "step": False, "tokens": 16384, "width": 2048, "symbols": 50021, "type": "bfloat16", "scale": 45.25, "padded": False},
        # Training in 32 bits, sizes that no vector load divides, short sequences filled up.
        {"name": "embed step 5003x1537 f32", "op": "embed", "step": True, "tokens": 5003, "width": 1537, "symbols": 10007, "type": "float32", "scale": 1.0, "padded": True},
        # Training of a medium model: most symbols of the table do not occur.
        {"name": "embed step 8192x1024 f16", "op": "embed", "step": True, "tokens": 8192, "width": 1024, "symbols": 32768, "type": "float16", "scale": 32.0, "padded": True},
        # Training of a large model on a large batch: the longest step.
        {"name": "embed step 65536x4096 bf16", "op": "embed", "step": True, "tokens": 65536, "width": 4096, "symbols": 131072, "type": "bfloat16", "scale": 1.0, "padded": False},
        # The log-probabilities of a few given symbols: latency counts.
        {"name": "entropy 7x1000 f32", "op": "entropy", "step": False, "tokens": 7, "width": 256, "symbols": 1000, "type": "float32", "padded": False},
        # Scoring of a few answers over an odd number of symbols: the table is read once for few rows.
        {"name": "entropy 64x50021 bf16", "op": "entropy", "step": False, "tokens": 64, "width": 2048, "symbols": 50021, "type": "bfloat16", "padded": False},
        # Evaluation of a batch.
        {"name": "entropy 8192x32768 f16", "op": "entropy", "step": False, "tokens": 8192, "width": 2048, "symbols": 32768, "type": "float16", "padded": True},
        # Training in 32 bits, odd sizes.
        {"name": "entropy step 1000x10007 f32", "op": "entropy", "step": True, "tokens": 1000, "width": 513, "symbols": 10007, "type": "float32", "padded": True},
        # Training of a small model with 16-bit floats and a scaled loss.
        {"name": "entropy step 2048x50021 f16", "op": "entropy", "step": True, "tokens": 2048, "width": 1024, "symbols": 50021, "type": "float16", "padded": True},
        # Training of a large model: the largest call.
        {"name": "entropy step 8192x131072 bf16", "op": "entropy", "step": True, "tokens": 8192, "width": 4096, "symbols": 131072, "type": "bfloat16", "padded": False},
    ]  # fmt: skip


def _between(rng, low, high):
    """A whole number of the range, spread over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind, step, padded = rng.choice(list(_TYPES)), rng.random() < 0.6, rng.random() < 0.5
    if rng.random() < 0.5:
        while True:
            tokens, width, symbols = _between(rng, 1, 65536), _between(rng, 64, 8192), _between(rng, 500, 200_000)
            width = max(64, width // 64 * 64) if rng.random() < 0.5 else width
            if (tokens + symbols) * width * (2 if kind == "float32" else 1) <= 65536 * 3 * 4096:
                break
        scale = rng.choice([1.0, round(math.sqrt(width), 3)])
        return {"op": "embed", "step": step, "tokens": tokens, "width": width, "symbols": symbols, "type": kind, "scale": scale, "padded": padded}
    while True:
        tokens, width, symbols = _between(rng, 1, 16384), _between(rng, 64, 8192), _between(rng, 500, 200_000)
        width = max(64, width // 64 * 64) if rng.random() < 0.7 else width
        work = tokens * width * symbols * (8 if kind == "float32" else 1)
        if work <= 8192 * 4096 * 131072 // 4 and tokens * symbols <= 8192 * 65536:
            break
    return {"op": "entropy", "step": step, "tokens": tokens, "width": width, "symbols": symbols, "type": kind, "padded": padded}


# ----------------------------------------------------------------------------- inputs


def _frequencies(symbols):
    """How often symbols occur in texts: in inverse proportion to their rank, but for the first few."""
    p = 1.0 / (np.arange(symbols) + 2.7)
    return p / p.sum()


def _tokens(case, g):
    """Symbols by their frequencies."""
    upto = torch.as_tensor(np.cumsum(_frequencies(case["symbols"])), device="cuda")
    at = torch.rand(case["tokens"], generator=g, device="cuda", dtype=torch.float64)
    return torch.searchsorted(upto, at).clamp_(max=case["symbols"] - 1)


def _filled(case, g):
    """The positions behind the ends of sequences: about an eighth, in runs."""
    n = case["tokens"]
    at = torch.arange(n, device="cuda")
    ends = 48 + 16 * torch.rand((n + 63) // 64, generator=g, device="cuda")
    return (at % 64) >= ends[at // 64]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    kind, n, width, symbols = _TYPES[case["type"]], case["tokens"], case["width"], case["symbols"]
    tokens = _tokens(case, g)
    filled = _filled(case, g) if case["padded"] else None
    # rows of a table as they are after training: some symbols' longer than others'
    weight = (randn(symbols, width) * (0.02 * torch.exp(0.3 * randn(symbols, 1)))).to(kind)
    if case["op"] == "embed":
        state = {"op": "embed", "step": case["step"], "tokens": tokens, "weight": weight, "scale": case["scale"], "padding": None}
        if case["padded"]:
            state["tokens"], state["padding"] = torch.where(filled, PADDING, tokens), PADDING
        if case["step"]:
            state["dy"] = (0.05 * randn(n, width)).to(kind)
        return state
    # activations that point, some more and some less, at the symbol that follows
    aim = weight[tokens].float()
    x = (randn(n, width) + 8.0 * torch.rand(n, 1, generator=g, device="cuda") * aim / aim.norm(dim=-1, keepdim=True)).to(kind)
    target = torch.where(filled, IGNORED, tokens) if case["padded"] else tokens
    # (gradients of 16-bit floats need a loss that is scaled up)
    dloss = torch.full((), 2.0**15 if kind == torch.float16 else 1.0, device="cuda")
    return {"op": "entropy", "step": case["step"], "x": x, "weight": weight, "target": target, "dloss": dloss}


# ----------------------------------------------------------------------------- plain forms


def _plain_embedding(tokens, weight, scale):
    return (weight[tokens].float() * scale).to(weight.dtype)


def _plain_embedding_backward(dy, tokens, symbols, scale, padding):
    d = dy.float()
    if padding is not None:
        d = torch.where((tokens == padding)[:, None], 0.0, d)
    total = torch.zeros(symbols, dy.shape[-1], device=dy.device).index_add_(0, tokens, d)
    return (total * scale).to(dy.dtype)


def _plain_entropy(x, weight, target, dloss):
    """Each position's loss, and log-sum-exp; with `dloss`, the mean loss and the gradients of dloss times it."""
    z = x.float() @ weight.float().t()
    top = z.max(-1, keepdim=True).values
    p = torch.exp(z - top)
    total = p.sum(-1, keepdim=True)
    lse = (top + torch.log(total)).squeeze(-1)
    given = target != IGNORED
    at = torch.where(given, target, 0)[:, None]
    loss = torch.where(given, lse - z.gather(1, at).squeeze(-1), 0.0)
    if dloss is None:
        return loss, lse
    count = given.sum().clamp(min=1)
    d = p / total
    d.scatter_add_(1, at, torch.full_like(total, -1.0))
    d *= torch.where(given, dloss / count, 0.0)[:, None]
    return loss.sum() / count, lse, (d @ weight.float()).to(x.dtype), (d.t() @ x.float()).to(weight.dtype)


def run(state):
    if own:
        import triturus_b200 as tb
    if state["op"] == "embed":
        tokens, weight, scale, padding = (state[n] for n in ("tokens", "weight", "scale", "padding"))
        y = tb.embedding(tokens, weight, scale=scale, padding_idx=padding) if own else _plain_embedding(tokens, weight, scale)
        if not state["step"]:
            return {"y": y}
        if own:
            dweight = tb.embedding_backward(state["dy"], tokens, weight.shape[0], scale=scale, padding_idx=padding)
        else:
            dweight = _plain_embedding_backward(state["dy"], tokens, weight.shape[0], scale, padding)
        return {"y": y, "dweight": dweight}
    x, weight, target = state["x"], state["weight"], state["target"]
    if not own:
        names = ("loss", "lse", "dx", "dweight")
        return dict(zip(names, _plain_entropy(x, weight, target, state["dloss"] if state["step"] else None)))
    if not state["step"]:
        loss, lse = tb.linear_cross_entropy(x, weight, target, ignore_index=IGNORED, reduction="none", return_lse=True)
        return {"loss": loss, "lse": lse}
    loss, lse = tb.linear_cross_entropy(x, weight, target, ignore_index=IGNORED, return_lse=True)
    dx, dweight = tb.linear_cross_entropy_backward(state["dloss"], x, weight, target, lse, ignore_index=IGNORED)
    return {"loss": loss, "lse": lse, "dx": dx, "dweight": dweight}


# ----------------------------------------------------------------------------- definitions in 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "embed":
        weight = state["weight"].double().requires_grad_(case["step"])
        y = torch.nn.functional.embedding(state["tokens"], weight, padding_idx=state["padding"]) * state["scale"]
        if not case["step"]:
            return {"y": y}
        (dweight,) = torch.autograd.grad(y, weight, state["dy"].double())
        return {"y": y.detach(), "dweight": dweight}
    x, weight = (state[n].double() for n in ("x", "weight"))
    target, width = state["target"], max(1, 2**28 // case["tokens"])  # (pieces of the table, for the memory's sake)
    pieces = [slice(b, b + width) for b in range(0, case["symbols"], width)]
    lse = torch.logsumexp(torch.stack([torch.logsumexp(x @ weight[s].t(), -1) for s in pieces]), 0)
    given = (target != IGNORED).nonzero().squeeze(-1)
    aim = weight[target[given]]
    loss = torch.zeros_like(lse)
    loss[given] = lse[given] - torch.linalg.vecdot(x[given], aim)
    if not case["step"]:
        return {"loss": loss, "lse": lse}
    share = 1.0 / max(1, given.numel())
    g = float(state["dloss"]) * share
    dx, dweight = torch.zeros_like(x), torch.zeros_like(weight)
    for s in pieces:
        p = torch.exp(x[given] @ weight[s].t() - lse[given, None])
        dx[given] += g * (p @ weight[s])
        dweight[s] = g * (p.t() @ x[given])
    dx[given] -= g * aim
    dweight.index_add_(0, target[given], x[given], alpha=-g)
    return {"loss": loss.sum() * share, "lse": lse, "dx": dx, "dweight": dweight}


# ----------------------------------------------------------------------------- work


def work(case):
    """Inputs read once, outputs written once.

    Lookup: the rows that occur are read, a row is written for each token, and the gradient reads one for each token and writes the
    table.  Cross entropy: one product of the activations and the table, two more for the gradients (2 operations for each of
    tokens x width x symbols); that the logits are not kept and have to be computed twice is not counted."""
    n, width, symbols, e = case["tokens"], case["width"], case["symbols"], _TYPES[case["type"]].itemsize
    if case["op"] == "embed":
        occur = float((1.0 - (1.0 - _frequencies(symbols)) ** n).sum())
        if not case["step"]:
            return {"bytes": int((n + occur) * width * e) + 8 * n, "flops": n * width}
        return {"bytes": int((2 * n + occur + symbols) * width * e) + 8 * n, "flops": 2 * n * width}
    nbytes = (n + symbols) * width * e + 12 * n
    return {"bytes": (2 if case["step"] else 1) * nbytes, "flops": (6 if case["step"] else 2) * n * width * symbols}

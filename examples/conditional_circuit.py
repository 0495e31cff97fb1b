"""A small conditional circuit, trained and sampled from with the operators of this package.

A network reads features and gives the log-probabilities of a layer of hidden states; a sum layer of a circuit (`lm2exp`) mixes them into the
log-probabilities of symbols:

    s[k] = relu(layer_norm(x[k] W0)) W1,   b[j, k] = log_softmax(s[k])_j,   out[v, k] = log sum_j a[v, j] exp b[j, k],   a = softmax_v(A)

Training follows the gradient of -mean_k out[y_k, k], clipped by its norm over all parameters; an answer is a symbol drawn from out[:, k].

    python examples/conditional_circuit.py [steps]
"""

from __future__ import annotations

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import triturus_b200 as tb  # noqa: E402

FEATURES, HIDDEN, STATES, SYMBOLS, BATCH = 64, 256, 128, 1000, 512


class Product(torch.autograd.Function):
    """a @ b through the package's matrix product."""

    @staticmethod
    def forward(ctx, a, b):
        ctx.save_for_backward(a, b)
        return tb.mm(a, b)

    @staticmethod
    def backward(ctx, g):
        a, b = ctx.saved_tensors
        g = g.contiguous()
        return tb.mm(g, b.t().contiguous()), tb.mm(a.t().contiguous(), g)


class SumLayer(torch.autograd.Function):
    """out[v, k] = log sum_j a[v, j] exp b[j, k], with d out[v, k] / d a[v, j] = exp(b[j, k] - out[v, k])
    and d out[v, k] / d b[j, k] = a[v, j] exp(b[j, k] - out[v, k])."""

    @staticmethod
    def forward(ctx, a, b):
        out = tb.lm2exp(a[None], b[None])[0]
        ctx.save_for_backward(a, b, out)
        return out

    @staticmethod
    def backward(ctx, g):
        a, b, out = ctx.saved_tensors
        top = b.amax(0, keepdim=True)
        e, g = torch.exp(b - top), g * torch.exp(top - out)
        return tb.mm(g, e.t().contiguous()), e * tb.mm(a.t().contiguous(), g)


class ConditionalCircuit:
    def __init__(self, seed: int = 0, device: str = "cuda"):
        g = torch.Generator().manual_seed(seed)
        randn = lambda *shape: torch.randn(*shape, generator=g)  # noqa: E731
        first = [randn(FEATURES, HIDDEN) / FEATURES**0.5, torch.ones(HIDDEN), torch.zeros(HIDDEN), randn(HIDDEN, STATES) / HIDDEN**0.5, 0.1 * randn(SYMBOLS, STATES)]
        self.parameters = [p.to(device).requires_grad_() for p in first]

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        """Log-probabilities [SYMBOLS, len(x)]."""
        w0, gain, shift, w1, emission = self.parameters
        h = tb.layer_norm(Product.apply(x, w0), gain, shift)
        b = torch.log_softmax(Product.apply(torch.relu(h), w1), dim=-1).t().contiguous()
        return SumLayer.apply(torch.softmax(emission, dim=0), b)

    def answer(self, x: torch.Tensor, noise: torch.Tensor, **filters):
        """A symbol for each row of x and its log-probability under the filtered distribution."""
        with torch.no_grad():
            return tb.sample(self(x).t(), noise, **filters, return_logprob=True)


def batch(g: torch.Generator, device: str = "cuda"):
    """Features around one of 40 centres, and a symbol that the centre gives two thirds of the time."""
    centres = torch.randn(40, FEATURES, generator=torch.Generator().manual_seed(1))
    which = torch.randint(40, (BATCH,), generator=g)
    x = centres[which] + 0.3 * torch.randn(BATCH, FEATURES, generator=g)
    y = torch.where(torch.rand(BATCH, generator=g) < 2 / 3, which * 25, torch.randint(SYMBOLS, (BATCH,), generator=g))
    return x.to(device), y.to(device), (which * 25).to(device)


def main(steps: int = 200, seed: int = 0) -> dict:
    model = ConditionalCircuit(seed)
    optimizer = torch.optim.Adam(model.parameters, lr=3e-2)
    g = torch.Generator().manual_seed(seed)
    losses, norms = [], []
    for _ in range(steps):
        x, y, _ = batch(g)
        loss = -model(x).gather(0, y[None]).mean()
        optimizer.zero_grad()
        loss.backward()
        norms.append(tb.clip_grad_norm_([p.grad for p in model.parameters], 0.5))
        optimizer.step()
        losses.append(loss.detach())
    x, _, centre = batch(g)
    noise = torch.empty(BATCH, SYMBOLS, device="cuda").exponential_()
    greedy, _ = model.answer(x, noise, temperature=0.0)
    token, logprob = model.answer(x, noise, temperature=0.8, top_k=50, top_p=0.95)
    tb.check_status()
    return {
        "losses": torch.stack(losses).tolist(),
        "norms": torch.stack(norms).tolist(),
        "greedy": float((greedy == centre).float().mean()),
        "token": token.cpu(),
        "logprob": logprob.cpu(),
    }


if __name__ == "__main__":
    got = main(int(sys.argv[1]) if len(sys.argv) > 1 else 200)
    print(f"loss {got['losses'][0]:.3f} -> {got['losses'][-1]:.3f}, most probable symbol right for {100 * got['greedy']:.0f} %")

"""GPU: the example trains and samples a circuit with layer_norm, clip_grad_norm_ and sample beside lm2exp and mm."""

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


def _example():
    path = Path(__file__).resolve().parent.parent / "examples" / "conditional_circuit.py"
    spec = importlib.util.spec_from_file_location("conditional_circuit", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_example_learns_and_answers():
    ex = _example()
    got = ex.main(steps=80)
    # the first loss is that of almost equal symbols, log 1000; the centres alone explain two thirds of them
    assert abs(got["losses"][0] - torch.tensor(float(ex.SYMBOLS)).log()) < 0.5
    assert got["losses"][-1] < 0.8 * got["losses"][0]
    assert got["greedy"] > 0.5
    assert all(n > 0 for n in got["norms"])
    assert int(got["token"].min()) >= 0 and int(got["token"].max()) < ex.SYMBOLS
    assert float(got["logprob"].max()) <= 1e-5 and bool(got["logprob"].isfinite().all())


def test_example_gradients_against_torch():
    """All of the model's gradients against the same formulas in float64 through torch's autograd.  3xTF32 products and logarithms are good to
    some 1e-6 of the terms, and each layer adds its own: 1e-3 of the largest element bounds them by far."""
    ex = _example()
    model = ex.ConditionalCircuit(3)
    x, y, _ = ex.batch(torch.Generator().manual_seed(5))
    (-model(x).gather(0, y[None]).mean()).backward()
    w0, gain, shift, w1, emission = [p.detach().double().requires_grad_() for p in model.parameters]
    u = x.double() @ w0
    h = (u - u.mean(-1, keepdim=True)) / torch.sqrt(u.var(-1, unbiased=False, keepdim=True) + 1e-5) * gain + shift
    b = torch.log_softmax(torch.relu(h) @ w1, dim=-1).t()
    out = torch.log(torch.softmax(emission, dim=0) @ torch.exp(b))
    (-out.gather(0, y[None]).mean()).backward()
    for mine, theirs in zip(model.parameters, (w0, gain, shift, w1, emission)):
        assert float((mine.grad.double() - theirs.grad).abs().max()) <= 1e-3 * float(theirs.grad.abs().max())

"""GPU: a small model of symbols with the operators together, as they would be used: embedding, layer_norm, matrix product, the cross entropy with
the embedding's own table, clipping, and symbols drawn from what it learned."""

import pytest
import torch

import triturus_b200 as tb

pytestmark = pytest.mark.gpu

V, D, IGNORE = 700, 96, -100


def model(table, gain, shift, tokens, target):
    h = tb.layer_norm(tb.embedding(tokens, table, scale=D**0.5, padding_idx=0), gain, shift)
    return tb.linear_cross_entropy(h, table, target, ignore_index=IGNORE), h


def parameters(kind):
    g = torch.Generator().manual_seed(4)
    table = (torch.randn(V, D, generator=g) * D**-0.5).to(kind).cuda()
    gain, shift = (1 + 0.1 * torch.randn(D, generator=g)).to(kind).cuda(), (0.1 * torch.randn(D, generator=g)).to(kind).cuda()
    tokens = torch.randint(V, (12, 40), generator=g).cuda()
    target = torch.randint(V, (12, 40), generator=g).cuda()
    tokens[:, 30:], target[:, 29:] = 0, IGNORE  # sequences that end early
    return [table, gain, shift], tokens, target


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_gradients_of_the_whole(kind):
    """Against float64 through torch's autograd, in the norm of each gradient.  float32: the norm and the products are good to some 1e-6 of their terms,
    1e-4 is far above it.  bfloat16: h, the embedding, d, and the gradients between the operators are rounded by 2^-9 (root mean square, a step being 2^-7) each, seven of
    them in a row, and two gradients of the table are added: 8 2^-8 = 3e-2 of the norms bounds their sum."""
    leaves, tokens, target = parameters(kind)
    mine = [p.clone().requires_grad_() for p in leaves]
    loss, _ = model(*mine, tokens, target)
    loss.backward()
    table, gain, shift = theirs = [p.double().requires_grad_() for p in leaves]
    e = torch.nn.functional.embedding(tokens, table, padding_idx=0) * D**0.5
    h = torch.nn.functional.layer_norm(e, (D,), gain, shift, 1e-5)
    want = torch.nn.functional.cross_entropy((h @ table.t()).flatten(0, 1), target.flatten(), ignore_index=IGNORE)
    want.backward()
    bound = 1e-4 if kind == torch.float32 else 3e-2
    assert abs(float(loss.detach()) - float(want.detach())) <= bound * float(want.detach())
    for a, b in zip(mine, theirs):
        assert a.grad.dtype == kind and float((a.grad.double() - b.grad).norm()) <= bound * float(b.grad.norm())
    norm = tb.clip_grad_norm_([p.grad for p in mine], 0.1)
    assert float(norm) > 0.1 and abs(float(tb.grad_norm([p.grad for p in mine])) - 0.1) <= 0.1 * 2.0**-8
    tb.check_status()


def test_log_probabilities_are_those_that_are_sampled_from():
    """-loss of a position is the logarithm of the probability with which `sample` draws its target."""
    leaves, tokens, target = parameters(torch.float32)
    with torch.no_grad():
        _, h = model(*leaves, tokens, target)
        logits = h.flatten(0, 1) @ leaves[0].t()
        noise = torch.empty_like(logits).exponential_()
        token, logprob = tb.sample(logits, noise, return_logprob=True)
        loss = tb.linear_cross_entropy(h, leaves[0], token.view(12, 40), reduction="none")
    assert torch.allclose(-loss.flatten(), logprob, rtol=0, atol=1e-3)


def test_a_captured_training_step():
    """Forward, backward and clipping as one graph, replayed on other symbols."""
    leaves, tokens, target = parameters(torch.bfloat16)
    static = [p.clone().requires_grad_() for p in leaves]

    def step():
        loss, _ = model(*static, tokens, target)
        grads = torch.autograd.grad(loss, static)
        return loss, *grads, tb.clip_grad_norm_(list(grads), 0.5)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    tokens.copy_(tokens.flip(0).clone())
    target.copy_(target.flip(0).clone())
    graph.replay()
    torch.cuda.synchronize()
    got = [t.detach().clone() for t in got]
    assert all(torch.equal(a, b.detach()) for a, b in zip(got, step()))
    tb.check_status()

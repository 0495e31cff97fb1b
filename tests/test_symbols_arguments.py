"""embedding and linear_cross_entropy take no fractions where they ask for whole numbers."""

import numpy as np
import pytest
import torch

import triturus_b200 as tb


def given():
    return torch.tensor([1, 2]), torch.randn(5, 8), torch.randn(2, 8), torch.zeros(2), torch.ones(())


def test_whole_numbers():
    tokens, weight, x, lse, one = given()
    for call, what in (
        (lambda: tb.embedding(tokens, weight, padding_idx=0.5), "padding_idx"),
        (lambda: tb.embedding_backward(x, tokens, 5, padding_idx=1.5), "padding_idx"),
        (lambda: tb.embedding_backward(x, tokens, 5.5), "symbols"),
        (lambda: tb.embedding_backward(x, tokens, torch.tensor(5.0)), "symbols"),
        (lambda: tb.linear_cross_entropy(x, weight, tokens, ignore_index=1.5), "ignore_index"),
        (lambda: tb.linear_cross_entropy(x, weight, tokens, ignore_index=None), "ignore_index"),
        (lambda: tb.linear_cross_entropy_backward(one, x, weight, tokens, lse, ignore_index=2.5), "ignore_index"),
    ):
        with pytest.raises(ValueError, match=what):
            call()


def test_whole_numbers_of_other_types():
    """They pass the checks: what is refused is the CPU tensor."""
    tokens, weight, x, lse, one = given()
    for call in (
        lambda: tb.embedding(tokens, weight, padding_idx=np.int64(1)),
        lambda: tb.embedding(tokens, weight, padding_idx=1.0),
        lambda: tb.embedding_backward(x, tokens, np.int32(5), padding_idx=True),
        lambda: tb.linear_cross_entropy(x, weight, tokens, ignore_index=np.int16(-1)),
        lambda: tb.linear_cross_entropy_backward(one, x, weight, tokens, lse, ignore_index=False),
    ):
        with pytest.raises(tb.NativeLibraryError, match="CUDA"):
            call()


@pytest.mark.gpu
def test_results_with_whole_numbers_of_other_types():
    tokens, weight, x, lse, one = (a.cuda() for a in given())
    assert torch.equal(tb.embedding_backward(x, tokens, np.int32(5), padding_idx=np.int64(1)), tb.embedding_backward(x, tokens, 5, padding_idx=1))
    tokens[0] = -1
    for kind in (np.int16, np.int64):
        assert torch.equal(tb.linear_cross_entropy(x, weight, tokens, ignore_index=kind(-1)), tb.linear_cross_entropy(x, weight, tokens, ignore_index=-1))
        got = tb.linear_cross_entropy_backward(one, x, weight, tokens, lse, ignore_index=kind(-1))
        want = tb.linear_cross_entropy_backward(one, x, weight, tokens, lse, ignore_index=-1)
        assert all(torch.equal(a, b) for a, b in zip(got, want))

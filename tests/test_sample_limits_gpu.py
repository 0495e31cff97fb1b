"""GPU: sample on rows around the limits of its kernels' forms, against the definition of test_sample_gpu."""

import pytest
import torch

import triturus_b200 as tb
from test_sample_gpu import BF16, F16, F32, check, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("symbols", [384_312, 384_316, 384_317, 384_325, 390_000, 393_208, 393_212, 393_217])
def test_longest_rows_in_shared_memory(symbols, kind):
    """Eight blocks with 48040 symbols each fill the shared memory that a block can have; longer rows are read again."""
    x, q = inputs(1, symbols, kind)
    check(x, q)
    check(x, q, top_k=40)
    check(x, q, top_p=0.9)


def test_longest_rows_of_a_batch():
    x, q = inputs(18, 390_000)
    check(x, q, top_k=20, top_p=0.7, temperature=0.6)


def test_nan_in_long_rows_at_any_temperature():
    x, q = inputs(200, 40_000)
    x[7, 123] = float("nan")
    x[9, 39_999] = float("nan")
    x[11, 20_000] = float("inf")
    for temperature in (1.0, 1e30, 1e38, 3e38):
        token, logprob = tb.sample(x, q, temperature=temperature, return_logprob=True)
        for i in (7, 9):
            assert int(token[i]) == -1 and bool(logprob[i].isnan())
        assert int((token < 0).sum()) == 2 and int(logprob.isnan().sum()) == 2

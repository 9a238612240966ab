"""Log probabilities (yskn_b200_token_logprobs) of more tokens a row than a CTA has threads, and more of the largest than
the row has tokens, against 64-bit sums within the bound of test_gpu_token_logprobs.py."""
import numpy as np
import pytest

from test_gpu_token_logprobs import call, check, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V,M,n", [(7, 3, 257), (3001, 2, 256), (3001, 2, 300), (50257, 1, 1000), (151936, 2, 513),
                                   (20011, 320, 290)])
def test_more_tokens_than_threads(cuda, V, M, n):
    """One part a row and several; the logits of the first 256 tokens are asked for ahead of the row, the others not."""
    x = rows(V + n, M, V)
    tokens = np.random.default_rng(n).integers(0, V, (M, n))
    tokens[:, ::7] = x.argmax(1)[:, None]  # the same token again
    tokens[:, -1] = V - 1
    check(cuda, x, tokens, 3)
    assert np.array_equal(call(cuda, x, tokens, 0)[0], call(cuda, x, tokens, 3)[0])


@pytest.mark.parametrize("k", [1, 8, 24, 25, 32])
@pytest.mark.parametrize("V", [1, 2, 7, 24, 25, 31, 130])
def test_more_of_the_largest_than_tokens(cuda, V, k):
    x = rows(V + k, 3, V)
    x[1, V // 2:] = -np.inf
    x[1, 0] = 1.0
    x[2, :] = 2.5
    check(cuda, x, [[0, V - 1]] * 3, k)

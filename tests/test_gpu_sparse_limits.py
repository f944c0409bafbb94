"""Sparse decode and log probabilities at the ends of what their arguments may be."""
import numpy as np
import pytest

import velokv
from test_gpu_logprobs import run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,vocab", [(2, 100), (3, 20000), (2, 70000)])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_extreme_scales(ctx, dtype, rows, vocab):
    """The largest scale leaves the row's largest logits alone, equally likely; the least makes all logits equal.
    log n is one fp32 logarithm and product from what is returned: 2^-22 relative is four roundings."""
    x = np.zeros((rows, vocab), dtype)
    x[:, 1::2] = 1
    x[:, 50] = -np.inf
    tokens = np.tile(np.array([0, 1, 50], np.int32), (rows, 1))
    for scale, n, first in ((2.35e38, vocab // 2, -np.inf), (1e-45, vocab - 1, -np.log(vocab - 1))):
        got = run(ctx, x, tokens, 2, scale=scale)
        want = np.array([first, -np.log(n), -np.inf])
        with np.errstate(invalid="ignore"):
            assert np.all((got["token_logprobs"] == want) | (np.abs(got["token_logprobs"] - want) <= 2.0 ** -22 * np.abs(want)))
        assert np.all(np.abs(got["entropy"] - np.log(n)) <= 2.0 ** -22 * np.log(n))
        assert np.array_equal(got["top_ids"], np.tile([1, 3], (rows, 1)))

"""Draws whose borders fall exactly between two candidates of the ranking: equal weights, of which a nucleus of a half keeps exactly half."""
import numpy as np
import pytest
from test_gpu_sample import _draw, draw64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [2, 8, 18, 56, 139, 256, 1000, 5000, 50257, 131072])
@pytest.mark.parametrize("top_p", [0.5, 0.25, 0.75, 0.125, 1 - 2.0**-10])
@pytest.mark.parametrize("top_k", [0, 16, 256, 700])
def test_nucleus_of_equal_logits(agpu, dev, n, top_p, top_k):
    """The sums of equal weights are exact on both sides, and so are the shares of them: before the first rank that is left out lies exactly top_p of the sum."""
    rng = np.random.default_rng(n)
    u = np.array([1 - 2.0**-24, 0.0, 0.5, *rng.random(3)], np.float32)
    for value, temperature in ((0.0, 1.0), (-3.5, 0.7), (1e4, 0.0)):
        x = np.full((len(u), n), value, np.float32)
        assert _draw(dev, x, u, temperature, top_k, top_p, 0.0) == draw64(x, u, temperature, top_k, top_p, 0.0)
        # some of them equal, the others without any weight beside them
        x[:, rng.permutation(n)[:n // 3]] -= 300.0
        assert _draw(dev, x, u, temperature, top_k, top_p, 0.0) == draw64(x, u, temperature, top_k, top_p, 0.0)

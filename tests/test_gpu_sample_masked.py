"""Sampling from a vocabulary of which a grammar or a mask leaves few tokens: the rest is -inf, or far
below every live logit."""
import numpy as np
import pytest

from tests._gpu import note
from tests.test_gpu_sample import run, want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("low", [-np.inf, -1e9, np.finfo(np.float32).min])
@pytest.mark.parametrize("vocab,live", [(700, 3), (50257, 1), (50257, 10), (151936, 12), (151936, 6000)])
def test_few_live_tokens(dev, vocab, live, low):
    """Cuts above, at and below the number of live tokens; more equal tokens than the kernels list."""
    note(f"sample {vocab}, {live} live, the rest {low}")
    rng = np.random.default_rng(vocab + live)
    rows = 3
    x = np.full((rows, vocab), low, np.float32)
    for r in range(rows):
        x[r, rng.choice(vocab, live, replace=False)] = 3 * rng.standard_normal(live)
    u = np.array([0.0, 0.41, 0.9999], np.float32)
    for c in (dict(), dict(top_k=50), dict(top_k=live), dict(top_k=max(live - 1, 1)), dict(top_k=live + 1, top_p=0.8),
              dict(top_p=0.95), dict(top_k=20000, top_p=0.9999999), dict(temperature=0.0), dict(top_k=50, min_p=0.05),
              dict(temperature=1e6, top_k=100)):
        np.testing.assert_array_equal(run(dev, x, u, **c), want(x, u, **c))

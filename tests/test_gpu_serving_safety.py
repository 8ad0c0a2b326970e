"""Serving operators where blocks, warps and calls meet one another: sampling rows whose blocks have little to read.

Sampled tokens are held to the definition's exactly (whole-number weights).
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_serving import dev, sample  # noqa: E402


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("b,v", [(3000, 4097), (1500, 8200), (1100, 16385), (600, 32769)])
def test_sample_rows_of_many_short_blocks(um, backend, half, b, v):
    """Thousands of clusters whose blocks read a few thousand logits each and start at different times: the largest
    logit, wherever it lies, reaches every block, and equal logits are drawn exactly."""
    rng = np.random.default_rng(v)
    x = rng.standard_normal((b, v)).astype(np.float16 if half else np.float32)
    at = rng.integers(0, v, b)
    x[np.arange(b), at] = 9.0
    two = (at + 1 + rng.integers(0, v - 1, b)) % v
    x[np.arange(b), two] = 9.0
    u = rng.random(b).astype(np.float32)
    xd = dev(x)
    tok, prob, kept = sample(um, backend, xd, 0.0, u=u)
    assert np.array_equal(tok, np.minimum(at, two)) and (kept == 1).all() and (prob == 1).all()
    tok, prob, kept = sample(um, backend, xd, 1.0, min_p=0.9, u=u)  # the next logit is far below 9
    assert np.array_equal(tok, np.where(u < 0.5, np.minimum(at, two), np.maximum(at, two)))
    assert (kept == 2).all() and (prob == 0.5).all()

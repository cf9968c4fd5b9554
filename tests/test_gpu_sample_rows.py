"""bq_sample over rows that are read again: several cuts one after another, and
temperatures at the ends of fp32 (reference and tolerance: test_gpu_sample.py)."""
import numpy as np
import pytest

from test_gpu_sample import _check, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [20000, 131072])
def test_cuts_one_after_another(bq, vocab):
    """A top-p cut and the draw's cut over the same bins, in many rows at once, and a third cut for u = 1: the draws
    meet the definition, and equal calls give equal tokens."""
    rng = np.random.default_rng(vocab)
    rows = 48
    x = rng.standard_normal((rows, vocab)).astype(np.float32) * 0.7
    u = rng.random(rows).astype(np.float32)
    u[::5] = 1.0
    u[1::5] = np.float32(1) - np.float32(2) ** -24
    print(f"sample cuts in turn, vocab {vocab}", flush=True)
    for k, p, t in ((0, 0.9, 1.0), (0, 0.999, 3.0), (vocab // 2, 0.6, 1.0), (0, 0.3, 1.0)):
        got = _check(bq, x, u, t, k, p, 0.0)
        for _ in range(3):
            assert np.array_equal(got, _run(bq, x, u, t, k, p, 0.0)), (k, p, t)

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


@pytest.mark.parametrize("vocab", [300, 20000, 131072])
def test_endless_temperature(bq, vocab):
    """Temperature inf: every token that is not -inf is as likely as the others, in the order of the logits."""
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((8, vocab)).astype(np.float32)
    x[:, rng.random(vocab) < 0.9] = -np.inf
    x[4:, 7:] = -np.inf   # few tokens
    u = np.array([0.0, 0.25, 0.6, 0.99] * 2, np.float32)
    for k, p in ((0, 1.0), (0, 0.5), (5, 1.0)):
        got = _run(bq, x, u, np.inf, k, p)
        for r in range(8):
            order = np.argsort(-x[r], kind="stable")[: int(np.isfinite(x[r]).sum())]
            if len(order) == 0:  # a row of -inf
                assert got[r] == 0
                continue
            n = len(order) if k == 0 else min(k, len(order))
            n = max(1, int(np.ceil(p * n)))
            at = int(np.floor(float(u[r]) * n))
            near = [order[i] for i in (at - 1, at, at + 1) if 0 <= i < n and abs(i - float(u[r]) * n + 0.5) <= 0.5 + 1e-4 * n]
            assert got[r] in near, (k, p, r, got[r], near)


@pytest.mark.parametrize("temp", [1e-37, 1e-38, 1e-39, 1e-44])
@pytest.mark.parametrize("tied", [3, 100, 3000])
def test_tiny_temperature(bq, temp, tied):
    """Next to no temperature: the tokens tied at the maximum share the mass."""
    vocab = 50000
    rng = np.random.default_rng(tied)
    x = rng.standard_normal((4, vocab)).astype(np.float32)
    at = np.sort(rng.choice(vocab, tied, replace=False))
    x[:, at] = 9.0
    u = ((np.array([0, tied // 3, tied // 2, tied - 1]) + 0.5) / tied).astype(np.float32)
    for p in (1.0, 0.9999):
        got = _run(bq, x, u, temp, 0, p)
        assert (got == at[[0, tied // 3, tied // 2, tied - 1]]).all(), (p, got)

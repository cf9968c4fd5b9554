"""bq_sample against the definition in 64 bits (tests/serve_ref.py: sample_ok).

Tolerance: a mass is exp of (logit - max) / temperature in fp32 (its argument,
at most 40 here where the mass counts, rounded to 2^-24: 2.4e-6 of a mass of
e^-40, 1e-7 of one that matters), sums are exact or, for the row's mass, fp32
per slice.  A draw or a cut may move by eps = 2e-6 of the mass.
"""
import ctypes

import numpy as np
import pytest
import torch

import serve_ref as R

pytestmark = pytest.mark.gpu


def _run(bq, logits, u, temp=None, k=None, p=None, mp=None):
    rows = logits.shape[0]
    f = lambda v, dt: None if v is None else torch.from_numpy(np.broadcast_to(np.asarray(v, dt), (rows,)).copy()).cuda()
    out = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    g = torch.from_numpy(logits).cuda() if isinstance(logits, np.ndarray) else logits
    bq.Sampler(g, out, f(u, np.float32), f(temp, np.float32), f(k, np.int32), f(p, np.float32), f(mp, np.float32)).run()
    return out.cpu().numpy()


def _check(bq, logits, u, temp=1.0, k=0, p=1.0, mp=0.0):
    got = _run(bq, logits, u, temp, k, p, mp)
    rows = logits.shape[0]
    full = lambda v, dt=np.float32: np.broadcast_to(np.asarray(v, dt), (rows,))
    for r in range(rows):
        assert R.sample_ok(logits[r], float(full(u)[r]), float(full(temp)[r]), int(full(k, np.int32)[r]),
                           float(full(p)[r]), float(full(mp)[r]), int(got[r])), (r, got[r])
    return got


def _peaked(seed, rows, vocab):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, vocab)).astype(np.float32) * 1.5
    for r in range(rows):
        x[r, rng.choice(vocab, min(40, vocab), replace=False)] += rng.uniform(4, 12, min(40, vocab)).astype(np.float32)
    return x


@pytest.mark.parametrize("vocab", [1, 3, 255, 8192, 8196, 32000, 131072, 262148])
def test_vocabularies_and_rules(bq, vocab):
    rng = np.random.default_rng(vocab)
    x = _peaked(vocab, 6, vocab)
    ld = vocab + 3
    buf = np.full((6, ld), 1e30, np.float32)   # what lies between rows is not read
    buf[:, :vocab] = x
    print(f"sample vocab {vocab}", flush=True)
    for k, p, mp, t in ((0, 1.0, 0.0, 1.0), (1, 1.0, 0.0, 1.0), (5, 1.0, 0.0, 0.7), (50, 0.9, 0.0, 0.8), (0, 0.9, 0.0, 0.9),
                        (0, 0.5, 0.1, 1.2), (0, 1.0, 0.05, 1.0), (700, 0.99, 0.0, 1.5), (3000, 1.0, 0.0, 2.0),
                        (0, 0.9999, 0.0, 3.0), (40, 0.95, 0.02, 1.0)):
        u = rng.random(6).astype(np.float32)
        got = _run(bq, torch.from_numpy(buf).cuda()[:, :vocab], u, t, k, p, mp)
        for r in range(6):
            assert R.sample_ok(x[r], float(u[r]), t, k, float(np.float32(p)), float(np.float32(mp)), int(got[r])), (k, p, mp, t, r, got[r])


def test_rows_have_their_own_rules(bq):
    x = _peaked(3, 8, 50000)
    u = np.linspace(0, 0.999, 8).astype(np.float32)
    _check(bq, x, u, temp=[0.5, 1, 2, 0, -1, 0.01, 1, 1], k=[0, 3, 1, 5, 0, 0, 100000, -4],
           p=[0.9, 1, 1, 1, 0.5, 0.9, 0.3, 2.0], mp=[0, 0, 0, 0, 0, 0.5, 0, 1.5])
    # no rule at all
    _check(bq, x, u)
    assert (_run(bq, x, u) >= 0).all()


@pytest.mark.parametrize("flat", ["equal", "few", "slow"])
def test_flat_rows(bq, flat):
    """Rows whose kept tokens are many: equal logits (ties go to the lower index), two levels, a wide Gaussian."""
    rng = np.random.default_rng(5)
    vocab = 30000
    x = np.zeros((4, vocab), np.float32)
    if flat == "few":
        x = rng.integers(0, 3, (4, vocab)).astype(np.float32)
    elif flat == "slow":
        x = rng.standard_normal((4, vocab)).astype(np.float32) * 0.3
    u = np.array([0.0, 0.3, 0.77, 0.999], np.float32)
    for k, p, mp in ((0, 1.0, 0.0), (0, 0.5, 0.0), (1000, 1.0, 0.0), (20000, 0.7, 0.0), (0, 0.9, 0.3), (0, 0.0, 0.0)):
        got = _check(bq, x, u, 1.0, k, p, mp)
        if flat == "equal" and k == 1000:
            assert abs(got[1] - 300) <= 1


@pytest.mark.parametrize("vocab", [5000, 76721, 131072])
def test_cuts_near_the_end_of_the_head(bq, vocab):
    """Likely tokens bunched in neighbouring indices, and top-k, top-p and min-p that fall before, at and behind
    the last logit that the scan can vouch for (a hundred or two of the row)."""
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((6, vocab)).astype(np.float32) * 1.5
    for r in range(6):
        n = 8 * (r + 1)
        at = int(rng.integers(0, vocab - 200))
        x[r, at + rng.choice(200, n, replace=False)] += rng.uniform(4, 12, n).astype(np.float32)
    print(f"sample cuts vocab {vocab}", flush=True)
    for k in (12, 47, 100, 160, 250, 400, 0):
        for p, mp, t in ((1.0, 0.0, 0.8), (0.9, 0.0, 1.0), (0.97, 0.0, 2.0), (0.9999, 0.0, 1.0), (1.0, 1e-4, 1.0), (0.95, 3e-3, 2.0)):
            u = rng.random(6).astype(np.float32)
            _check(bq, x, u, t, k, p, mp)


@pytest.mark.parametrize("vocab", [700, 76721, 262148])
def test_no_filter(bq, vocab):
    """Temperature alone: draws among the likeliest tokens and far behind them, over a peaked and a flat row."""
    x = _peaked(vocab + 1, 12, vocab)
    x[6:] = np.random.default_rng(vocab).standard_normal((6, vocab)).astype(np.float32)
    u = np.array([0.0, 0.2, 0.6, 0.95, 0.99999, np.float32(1) - np.float32(2) ** -24] * 2, np.float32)
    print(f"sample unfiltered vocab {vocab}", flush=True)
    for t in (0.3, 1.0, 2.5):
        _check(bq, x, u, t)


def test_unusual_logits(bq):
    inf, nan = np.inf, np.nan
    vocab = 9000
    x = np.full((7, vocab), -inf, np.float32)
    x[1, 17] = 0
    x[2, [5, 8000]] = 1, 1
    x[3] = np.random.default_rng(1).standard_normal(vocab)
    x[3, ::2] = nan
    x[4, [100, 300]] = inf
    x[5] = nan
    x[6] = -3e38
    x[6, 4444] = 3e38
    u = np.full(7, 0.75, np.float32)
    got = _check(bq, x, u, 1.0, 0, 0.9, 0.0)
    assert list(got[[0, 1, 4, 5, 6]]) == [0, 17, 100, 0, 4444]
    assert got[2] == 8000 and got[3] % 2 == 1
    got = _run(bq, x, u, 0.0)
    assert list(got[[0, 1, 2, 4, 5, 6]]) == [0, 17, 5, 100, 0, 4444]
    # -0 and 0 are equal: the lower index first
    z = np.zeros((1, 64), np.float32)
    z[0, 0] = -0.0
    assert _run(bq, z, [0.0], 1.0, 1)[0] == 0
    # u at its ends
    y = _peaked(2, 3, 1000)
    _check(bq, y, np.array([0.0, np.float32(1) - np.float32(2) ** -24, 0.5], np.float32), 1.0, 20)


def test_draws_follow_the_distribution(bq):
    """u over an even grid: each token is drawn as often as its mass says, to one step of the grid."""
    row = np.array([2.0, 1.0, 0.0, -1.0] * 8, np.float32)
    n = 2000
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    got = _run(bq, np.repeat(row[None], n, 0), u, 1.0, 0, 1.0, 0.0)
    e = np.exp(row.astype(np.float64))
    want = e / e.sum() * n
    assert (np.abs(np.bincount(got, minlength=32) - want) <= 1.01).all()


def test_refusals(bq):
    L = bq.load()
    x = torch.zeros((2, 1000), device="cuda")
    out = torch.full((2,), -7, dtype=torch.int32, device="cuda")
    s = bq.Sampler(x, out, torch.zeros(2, device="cuda"))
    names = ["logits", "ld", "rows", "vocab", "temp", "k", "p", "mp", "u", "out", "work", "bytes"]

    def call(**change):
        a = dict(zip(names, s._args))
        a.update(change)
        return L.bq_sample(*[a[n] for n in names], bq._stream())

    E = bq.BQ_EINVAL
    for change in (dict(logits=None), dict(u=None), dict(out=None), dict(work=None), dict(bytes=8), dict(ld=998), dict(rows=-1),
                   dict(vocab=0), dict(logits=x.data_ptr() + 2), dict(work=s._keep[-1].data_ptr() + 4)):
        assert call(**change) == E, change
    assert call(vocab=(1 << 20) + 4, ld=(1 << 20) + 4) == bq.BQ_UNSUPPORTED
    assert call(rows=0) == bq.BQ_OK
    torch.cuda.synchronize()
    assert (out == -7).all()
    with pytest.raises(TypeError):
        bq.Sampler(x.half(), out, torch.zeros(2, device="cuda"))
    with pytest.raises(ValueError):
        bq.Sampler(x, out.long(), torch.zeros(2, device="cuda"))

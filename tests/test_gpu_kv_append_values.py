"""bq_append of rows whose values are not numbers or very small
(values: test_gpu_kv_append.py)."""
import pytest
import torch

import serve_ref as R
from test_gpu_kv_append import _rows

pytestmark = pytest.mark.gpu


def _append_raw(bq, kv, k, v, P=32):
    """k and v [rows, H * D] to tokens 0.. of one sequence, unnormed and unrotated; the cache."""
    rows, width = k.shape
    D, H = 64, width // 64
    cache = R.Pages(kv, H, D, P, 1, (rows + P - 1) // P, 3).cache(bq)
    pos = torch.arange(rows, dtype=torch.int32, device="cuda")
    bq.Append(cache, torch.zeros((rows, width), device="cuda"), k.cuda(), v.cuda(), pos, torch.empty((rows, width), device="cuda")).run()
    return cache, pos


@pytest.mark.parametrize("rows", [9, 1100])
@pytest.mark.parametrize("kv", ["bf16", "q8"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_is_no_number_stays_none(bq, kv, rows, bad):
    """A NaN or an infinity is not stored as a finite value (in q8 it takes its 32 values with it), and what
    stands beside it is stored as without it."""
    H, D = 2, 64
    k, v = _rows(1, rows, H * D), _rows(2, rows, H * D)
    clean = []
    for put in (False, True):
        if put:
            k[3, 5], v[3, 100], v[8, 33] = bad, bad, bad
        cache, pos = _append_raw(bq, kv, k, v)
        out = [torch.empty((rows, H * D), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        cache.read(pos, *out)
        clean.append([t.float().cpu() for t in out])
    for which, at in ((0, [(3, 5)]), (1, [(3, 100), (8, 33)])):
        same = torch.ones((rows, H * D), dtype=torch.bool)
        for r, c in at:
            assert not torch.isfinite(clean[1][which][r, c]), (which, r, c, clean[1][which][r, c])
            same[r, c // 32 * 32: c // 32 * 32 + 32] = False
        assert torch.equal(clean[0][which][same], clean[1][which][same])

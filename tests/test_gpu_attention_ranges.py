"""Attention over finite values, keys and queries of unusual size (helpers and
references: tests/serve_ref.py).

Tolerances, relative to sum_j p_j |v_j| of the output as in test_gpu_attention.py:
  converted q8 tiles (many rows): a value and a weight are 2^-11 each at most, the
    weight's underflow below 2^-9 of what the likeliest token's scale gives; fp32
    sums and the exponent's argument 2^-18 A:  tol = 2^-9 + 2^-18 A.
  tiles converted on the way: value and weight bf16, 2^-8 each:  2^-7 (1 + 2^-6) + 2^-18 A.
"""
import pytest
import torch

import serve_ref as R
from test_gpu_attention import _normal

pytestmark = pytest.mark.gpu


def _many_rows(bq, k, v, q, what, work="auto", scale=None):
    """T rows of 8 query heads a key-value head over T tokens; the worst error over its tolerance, by row."""
    T, H, D = k.shape
    Hq, P = 8 * H, 32
    pages = R.Pages("q8", H, D, P, 1, (T + P - 1) // P, 3)
    pages.put(0, k, v)
    out = torch.empty((T, Hq * D), device="cuda")
    att = bq.Attention(pages.cache(bq), q.cuda(), out, torch.tensor([T], dtype=torch.int32, device="cuda"), work=work, scale=scale)
    att.prefill()
    got = out.cpu().double().reshape(T, Hq, D)
    scale = D ** -0.5 if scale is None else scale
    ref, bound, A = R.attention(R.half_rows(q.reshape(T, Hq, D)), pages.kh[0], pages.v[0], torch.arange(T), scale)
    tol = (2.0 ** -9 if work == "auto" else 2.0 ** -7 * (1 + 2.0 ** -6)) + 2.0 ** -18 * A[..., None]
    ratio = ((got - ref).abs() / (tol * bound).clamp(min=1e-300)).amax((1, 2))
    print(f"  {what}: worst error / tolerance {ratio.max().item():.3f} at row {int(ratio.argmax())}", flush=True)
    assert torch.isfinite(out).all(), what
    assert (ratio <= 1).all(), (what, ratio.max().item())


def _inputs(T, H, D, seed):
    return _normal(seed, T, H, D), _normal(seed + 1, T, H, D), _normal(seed + 2, T, 8 * H * D) * 2


@pytest.mark.parametrize("work", ["auto", None])
@pytest.mark.parametrize("amplitude", [1e-3, 1e-5, 1e-6, 1e-20, 300.0, 1e6, 1e20])
def test_one_group_of_another_size(bq, amplitude, work):
    """32 dims of every token much smaller or larger than the others."""
    for D in (64, 128, 256):
        k, v, q = _inputs(288, 1, D, 51)
        v[:, :, 32:64] *= amplitude
        _many_rows(bq, k, v, q, f"group of {amplitude} D {D}", work)


@pytest.mark.parametrize("power", [10, 20, 40, 90])
def test_an_outlier_does_not_reach_rows_before_it(bq, power):
    """A large value late in a tile: the rows that cannot see it keep their precision."""
    k, v, q = _inputs(320, 1, 128, 61)
    v[63] *= 2.0 ** power
    v[200, :, 5] *= 2.0 ** power
    _many_rows(bq, k, v, q, f"outlier 2^{power}")


@pytest.mark.parametrize("first,then,far", [(40, -10, 60.0), (14, -25, 9.0), (100, 0, 60.0), (0, -60, 60.0)])
def test_large_values_with_little_weight(bq, first, then, far):
    """A tile of large values that later rows give next to no weight: what they do see stays exact."""
    T, D = 256, 128
    k, v, q = _inputs(T, 1, D, 71)
    v[:64] *= 2.0 ** first
    v[64:] *= 2.0 ** then
    # keys and queries share a direction with one sign in the first tile and the other after it
    k[:64, :, 0], k[64:, :, 0] = -far, far
    q.reshape(T, 8, D)[64:, :, 0] = 8.0
    _many_rows(bq, k, v, q, f"2^{first} then 2^{then}")


def test_values_of_zero(bq):
    """Groups, tokens and whole tiles of zeros."""
    k, v, q = _inputs(300, 2, 64, 81)
    v[:, 0, :32] = 0
    v[64:128] = 0
    v[5] = 0
    v[150:170] *= 1e-12
    _many_rows(bq, k, v, q, "zeros")


@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 20), (64, 0)])
@pytest.mark.parametrize("D,P", [(64, 16), (128, 64), (256, 32)])
def test_odd_sizes_behind_masks(bq, window, sinks, D, P):
    """Ragged chunks, unmapped pages, windows with sinks, pieces and strides, over values of mixed sizes, some
    tiles of each sequence ordinary; tokens that no row sees hold NaN scales."""
    H, Hq = 1, 8
    for rows, past, qt, ot in (([260, 5, 0, 70], [100, 400, 7, 0], torch.bfloat16, torch.bfloat16), ([270], [900], torch.float32, torch.float32)):
        lens = [a + b for a, b in zip(rows, past)]
        pages = R.Pages("q8", H, D, P, len(rows), max(lens) // P + 1, 7)
        for s, T in enumerate(lens):
            k, v = _normal(100 + s, T, H, D), _normal(200 + s, T, H, D)
            v[3::130] *= 1e12          # in every other tile or so
            v[150:160, :, 32:] *= 1e-9
            pages.put(s, k, v)
        holes = [(0, 0), (0, lens[0] // P // 2)]
        if window:  # nothing sees tokens from the sinks up to the first row's window
            for s, (r, T) in enumerate(zip(rows, lens)):
                t = torch.arange(sinks, max(sinks, T - r - window + 1))
                page = pages.table[s][t // P].long()
                for d in range(0, D, 32):
                    for value in (0, 1):
                        pages.raw.view(torch.bfloat16)[page, 0, R.addr_q8(P, D, t % P, torch.tensor(d), value)[1] // 2] = float("nan")
        for s, p in holes:
            pages.table[s, p] = -1
        total, pad = sum(rows), 8
        q = (_normal(9, total, Hq * D) * 2).to(qt)
        gq = torch.full((total, Hq * D + pad), float("nan"), dtype=qt, device="cuda")
        gq[:, : Hq * D] = q.cuda()
        out = torch.full((total, Hq * D + pad), float("nan"), dtype=ot, device="cuda")
        row0 = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], dtype=torch.int32, device="cuda")
        att = bq.Attention(pages.cache(bq), gq[:, : Hq * D], out[:, : Hq * D], torch.tensor(lens, dtype=torch.int32, device="cuda"),
                           window=window, sinks=sinks, row0=row0, max_rows=max(rows))
        att.prefill()
        assert torch.isnan(out[:, Hq * D:]).all()
        got = out[:, : Hq * D].cpu().double().reshape(total, Hq, D)
        qr = R.half_rows(q.float().reshape(total, Hq, D))
        first = 0
        for s, (r, T) in enumerate(zip(rows, lens)):
            hidden = torch.zeros(T, dtype=torch.bool)
            for hs, p in holes:
                if hs == s:
                    hidden[p * P:(p + 1) * P] = True
            ref, bound, A = R.attention(qr[first: first + r], pages.kh[s], pages.v[s], torch.arange(T - r, T), D ** -0.5, window, sinks, hidden)
            tol = 2.0 ** -9 + 2.0 ** -18 * A[..., None] + (2.0 ** -8 if ot == torch.bfloat16 else 0)
            ok = ((got[first: first + r] - ref).abs() <= tol * bound).all()
            assert torch.isfinite(got[first: first + r]).all() and ok, (s, r, T)
            first += r


def _one_hot(bq, kv, rows, q, k, v, what, prefill):
    """`rows` rows after T - rows tokens, whose scores are so far apart that each row's softmax is one token."""
    T, H, D = k.shape
    P, Hq = 32, q.shape[1] // D
    pages = R.Pages(kv, H, D, P, 1, (T + P - 1) // P, 5)
    pages.put(0, k, v)
    out = torch.empty((rows, Hq * D), device="cuda")
    att = bq.Attention(pages.cache(bq), q.cuda(), out, torch.tensor([T], dtype=torch.int32, device="cuda"))
    att.prefill() if prefill else att.decode()
    got = out.cpu().double().reshape(rows, Hq, D)
    q = q.reshape(rows, Hq, D)
    if prefill:
        q = R.bf16(q).double() if kv == "bf16" else R.half_rows(q)
    keys = pages.kh[0] if prefill else pages.k[0]
    scale = D ** -0.5
    ref, bound, A = R.attention(q.double(), keys, pages.v[0], torch.arange(T - rows, T), scale)
    s = scale * torch.einsum("rhd,thd->rht", q.double(), keys.repeat_interleave(Hq // H, 1))
    s.masked_fill_(torch.arange(T)[None, None] > torch.arange(T - rows, T)[:, None, None], -torch.inf)
    top = s.topk(2, -1).values
    assert ((top[..., 0] - top[..., 1])[1:] > 2.0 ** -18 * A[1:] + 100).all(), "the test's scores are too close"
    print(f"  {what}: finite {bool(torch.isfinite(got).all())}", flush=True)
    assert torch.isfinite(got).all(), what
    assert ((got - ref).abs() <= 2.0 ** -7 * bound)[1:].all(), what


@pytest.mark.parametrize("kv", ["bf16", "q8"])
@pytest.mark.parametrize("rows,prefill", [(300, True), (40, True), (5, False)])
@pytest.mark.parametrize("size,sign", [(1e4, 1), (1e4, -1), (1e6, 1), (1e6, -1), (1e8, 1), (1e8, -1), (1e16, 1)])
def test_scores_of_any_size(bq, kv, rows, prefill, size, sign):
    """Scores of 1e7 to 1e31, all a row's tokens on the same side of 0, still choose the largest."""
    T, D, Hq = max(rows, 150), 128, 8
    k, v, q = _normal(91, T, 1, D), _normal(92, T, 1, D), _normal(93, rows, Hq * D)
    # one dim decides, in a group of its own: 64 steps to a power of two, in a random order
    step = torch.randperm(T, generator=torch.Generator().manual_seed(1))
    k[:, 0, :32] = 0
    q.reshape(rows, Hq, D)[:, :, :32] = 0
    k[:, 0, 0] = sign * size * (1 + (step % 64).float() / 64) * 2.0 ** (step // 64 - 3).float()
    k[:, 0, 32:] *= 1e-3
    q.reshape(rows, Hq, D)[:, :, 0] = size * (1 + 2.0 ** -4 * torch.arange(Hq))
    _one_hot(bq, kv, rows, q, k, v, f"{kv} {rows} rows, scores {sign} * {size:.0e}^2", prefill)


@pytest.mark.parametrize("kv", ["bf16", "q8"])
@pytest.mark.parametrize("rows,prefill", [(300, True), (40, True), (5, False)])
def test_scores_far_below_zero(bq, kv, rows, prefill):
    """Scores of -1e31: rows that see tokens are not rows that see none."""
    test_scores_of_any_size(bq, kv, rows, prefill, 1e16, -1)


@pytest.mark.parametrize("rows,prefill", [(300, True), (40, True), (5, False)])
def test_zero_queries_with_a_tiny_scale(bq, rows, prefill):
    """Equal scores of 0, whatever the scale: the mean of what each row sees."""
    T, D, Hq, P = max(rows, 150), 128, 8, 32
    k, v = _normal(94, T, 1, D), _normal(95, T, 1, D)
    for kv in ("bf16", "q8"):
        pages = R.Pages(kv, 1, D, P, 1, (T + P - 1) // P, 5)
        pages.put(0, k, v)
        out = torch.empty((rows, Hq * D), device="cuda")
        att = bq.Attention(pages.cache(bq), torch.zeros((rows, Hq * D), device="cuda"), out,
                           torch.tensor([T], dtype=torch.int32, device="cuda"), scale=1e-20)
        att.prefill() if prefill else att.decode()
        got = out.cpu().double().reshape(rows, Hq, D)
        ref, bound, _ = R.attention(torch.zeros((rows, Hq, D), dtype=torch.float64), pages.k[0], pages.v[0],
                                    torch.arange(T - rows, T), 1e-20)
        assert torch.isfinite(got).all(), kv
        assert ((got - ref).abs() <= 2.0 ** -7 * (1 + 2.0 ** -6) * bound).all(), kv


@pytest.mark.parametrize("power", [-118, -60, 60, 100])
def test_keys_and_queries_of_opposite_size(bq, power):
    """Keys times 2^power and queries divided by it: the same scores."""
    T, D, Hq = 300, 128, 8
    k, v, q = _normal(96, T, 1, D), _normal(97, T, 1, D), _normal(98, T, Hq * D)
    for rows, prefill in ((300, True), (40, True), (5, False)):
        pages = R.Pages("q8", 1, D, 32, 1, (T + 31) // 32, 5)
        pages.put(0, k * 2.0 ** power, v)
        x = q[:rows] * 2.0 ** -power
        out = torch.empty((rows, Hq * D), device="cuda")
        att = bq.Attention(pages.cache(bq), x.cuda(), out, torch.tensor([T], dtype=torch.int32, device="cuda"))
        att.prefill() if prefill else att.decode()
        got = out.cpu().double().reshape(rows, Hq, D)
        xr = R.half_rows(x.reshape(rows, Hq, D)) if prefill else x.double().reshape(rows, Hq, D)
        ref, bound, A = R.attention(xr, (pages.kh if prefill else pages.k)[0], pages.v[0], torch.arange(T - rows, T), D ** -0.5)
        tol = (2.0 ** -7 * (1 + 2.0 ** -6) if prefill else 2.0 ** -16) + 2.0 ** -18 * A[..., None]
        assert torch.isfinite(got).all(), (power, rows)
        assert ((got - ref).abs() <= tol * bound).all(), (power, rows)

"""bq_attn_decode and bq_attn_prefill against 64-bit attention over what the
cache stands for (tests/serve_ref.py).  Bytes of the cache that hold no token
of a sequence are NaN throughout, so a masked place that counted would show.

Tolerances, relative to sum_j p_j |v_j| of the output (an error of the weights
moves the output by at most that times the weights' relative error, numerator
and denominator once each):
  fp32 decode: a weight as two bf16 parts (8 significant bits each) 2^-16; scores: fp32 sums of D <= 256
    exact products, 2^-24 per addition of at most A = scale sum |q_i k_i|, and
    the exponent's argument (x log2 e - m, at most 2 A log2 e) rounded once or
    twice: below 2^-19 A each way.  tol = 2^-16 + 2^-18 A.
  bf16 weights (prefill; decode with bf16 in and out): 2^-8 of a weight instead
    of 2^-16, and 2^-8 of a bf16 output: tol = 2^-7 (1 + 2^-6) + 2^-18 A.
Prefill takes q as bf16, and over a q8 cache q and keys as fp16 over a power of
two of their row, values as bf16: the reference rounds them the same.
"""
import ctypes

import numpy as np
import pytest
import torch

import serve_ref as R

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _normal(seed, *shape):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal(shape).astype(np.float32))


def _check(out, ref, bound, A, fine, what):
    tol = (2.0 ** -16 if fine else 2.0 ** -7 * (1 + 2.0 ** -6)) + 2.0 ** -18 * A[..., None]
    err = (out - ref).abs()
    assert torch.isfinite(out).all(), what
    ratio = (err / (tol * bound).clamp(min=1e-30)).max().item() if err.numel() else 0.0
    print(f"  {what}: worst error / tolerance {ratio:.3f}", flush=True)
    assert (err <= tol * bound).all(), (what, ratio)


def _decode(bq, kv, lens, rows, Hq, H, D, P, qt, ot, window=0, sinks=0, seed=1, work="auto", holes=(), max_len=None,
            pad=0, qscale=2.0):
    n = len(lens)
    max_pages = max(1, (max(lens) + P - 1) // P + 1)
    pages = R.Pages(kv, H, D, P, n, max_pages, seed)
    for s, T in enumerate(lens):
        if T:
            pages.put(s, _normal(seed * 100 + s, T, H, D), _normal(seed * 100 + 50 + s, T, H, D))
    for s, p in holes:
        pages.table[s, p] = -1
    cache = pages.cache(bq)
    q = (_normal(seed + 7, n * rows, Hq * D) * qscale).to(DT[qt])
    gq = torch.full((n * rows, Hq * D + pad), float("nan"), dtype=DT[qt], device="cuda")
    gq[:, : Hq * D] = q.cuda()
    out = torch.full((n * rows, Hq * D + pad), float("nan"), dtype=DT[ot], device="cuda")
    att = bq.Attention(cache, gq[:, : Hq * D], out[:, : Hq * D], torch.tensor(lens, dtype=torch.int32, device="cuda"),
                       window=window, sinks=sinks, work=work, max_len=max_len)
    att.decode()
    torch.cuda.synchronize()
    if pad:
        assert torch.isnan(out[:, Hq * D:]).all()
    got = out[:, : Hq * D].cpu().double().reshape(n, rows, Hq, D)
    for s, T in enumerate(lens):
        hidden = torch.zeros(T, dtype=torch.bool)
        for hs, p in holes:
            if hs == s:
                hidden[p * P:(p + 1) * P] = True
        if T:
            ref = R.attention(q[s * rows:(s + 1) * rows].double().reshape(rows, Hq, D), pages.k[s], pages.v[s],
                              torch.arange(T - rows, T), D ** -0.5, window, sinks, hidden)
        else:
            ref = [torch.zeros((rows, Hq, D), dtype=torch.float64)] * 2 + [torch.zeros((rows, Hq), dtype=torch.float64)]
        _check(got[s], *ref, not (qt == "bf16" and ot == "bf16") and ot != "bf16", f"decode seq {s} of {T} tokens")
    return out


@pytest.mark.parametrize("kv", ["bf16", "q8"])
@pytest.mark.parametrize("D,Hq,H,P", [(64, 8, 8, 16), (128, 32, 4, 64), (128, 6, 2, 16), (256, 7, 1, 32), (256, 2, 2, 256)])
def test_decode_lengths(bq, kv, D, Hq, H, P):
    _decode(bq, kv, [1, 0, 31, 32, 33, 65, 300, 129], 1, Hq, H, D, P, "f32", "f32", seed=D + Hq)


@pytest.mark.parametrize("kv", ["bf16", "q8"])
@pytest.mark.parametrize("qt,ot", [("f32", "bf16"), ("bf16", "f32"), ("bf16", "bf16")])
def test_decode_types_and_strides(bq, kv, qt, ot):
    for D in (64, 128, 256):
        _decode(bq, kv, [77, 200], 1, 8, 2, D, 32, qt, ot, seed=D, pad=8)


@pytest.mark.parametrize("kv", ["bf16", "q8"])
@pytest.mark.parametrize("rows", [2, 5, 8])
def test_verify_rows(bq, kv, rows):
    """Several new tokens; sequences shorter than the rows leave some with no token."""
    _decode(bq, kv, [3, 1, 0, 40, 333], rows, 24, 2, 128, 16, "f32", "f32", seed=rows)
    _decode(bq, kv, [70, 9], rows, 5, 5, 64, 64, "f32", "f32", seed=rows + 20)


@pytest.mark.parametrize("kv", ["bf16", "q8"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (32, 4), (100, 33), (64, 0), (500, 40)])
def test_decode_window_and_sinks(bq, kv, window, sinks):
    for rows in (1, 6):
        _decode(bq, kv, [5, 64, 410, 129], rows, 8, 2, 128, 16, "f32", "f32", window, sinks, seed=window + rows)
    _decode(bq, kv, [410, 222], 3, 8, 2, 64, 128, "bf16", "bf16", window, sinks, seed=window)


def test_decode_split_long(bq):
    """A long sequence beside short ones: split, unsplit and a small workspace agree with the reference."""
    for kv in ("bf16", "q8"):
        for work in ("auto", None):
            _decode(bq, kv, [5000, 17, 1300], 1, 8, 2, 128, 64, "f32", "f32", seed=3, work=work)
    small = torch.empty(2 * 3 * 2 * 16 * (128 + 2) + 7, device="cuda")  # two splits and a remainder
    _decode(bq, "bf16", [5000, 17, 1300], 1, 8, 2, 128, 64, "f32", "f32", seed=3, work=small)
    # more 32-token steps in a workgroup than it stages pages for at once
    _decode(bq, "q8", [66000], 1, 2, 1, 64, 16, "f32", "f32", seed=4, work=None)


@pytest.mark.parametrize("kv", ["bf16", "q8"])
@pytest.mark.parametrize("D,Hq,H,P", [(64, 6, 2, 16), (128, 16, 2, 64), (256, 3, 1, 32)])
def test_decode_split_shapes(bq, kv, D, Hq, H, P):
    """Pieces and their join at each head width: several new tokens, windows wider than a piece, unmapped pages,
    sequences that fill only the first piece or none."""
    lens = [1500, 1, 0, 1090, 33]
    _decode(bq, kv, lens, 1, Hq, H, D, P, "f32", "f32", seed=D + 2)
    _decode(bq, kv, lens, 5, Hq, H, D, P, "bf16", "bf16", seed=D + 3)
    _decode(bq, kv, lens, 3, Hq, H, D, P, "f32", "bf16", 1200, 40, seed=D + 4)
    _decode(bq, kv, lens, 1, Hq, H, D, P, "f32", "f32", seed=D + 5, holes=[(0, 0), (0, 12), (3, 9)])


def test_decode_peaked_scores(bq):
    """Scores tens apart: the running maximum moves often; and far below the first ones."""
    for kv in ("bf16", "q8"):
        _decode(bq, kv, [700, 90], 1, 8, 2, 128, 32, "f32", "f32", seed=5, qscale=25.0)


def test_decode_unmapped_pages(bq):
    _decode(bq, "bf16", [200, 40, 16], 2, 8, 2, 128, 16, "f32", "f32", seed=6, holes=[(0, 3), (0, 11), (2, 0)])
    _decode(bq, "q8", [200, 300], 1, 8, 2, 64, 64, "f32", "f32", seed=7, holes=[(0, 0), (1, 4)])


def test_decode_clamps_length(bq):
    """kv_len beyond max_len or the table, and negative, is clamped."""
    H, D, P = 1, 64, 16
    pages = R.Pages("bf16", H, D, P, 3, 4, 8)
    for s in range(3):
        pages.put(s, _normal(s, 64, H, D), _normal(9 + s, 64, H, D))
    cache = pages.cache(bq)
    q = _normal(20, 3, 2 * D)
    out = torch.empty((3, 2 * D), device="cuda")
    for max_len, seen in ((64, [64, 64, 0]), (40, [40, 40, 0])):
        bq.Attention(cache, q.cuda(), out, torch.tensor([1 << 30, 64, -5], dtype=torch.int32, device="cuda"),
                     max_len=max_len).decode()
        got = out.cpu().double().reshape(3, 1, 2, D)
        for s in range(3):
            if seen[s] == 0:
                assert (got[s] == 0).all()
                continue
            # the row's position is the clamped length's last token
            ref = R.attention(q[s: s + 1].double().reshape(1, 2, D), pages.k[s], pages.v[s], [seen[s] - 1], D ** -0.5)
            _check(got[s], *ref, True, f"clamped {max_len} seq {s}")


def _prefill(bq, kv, rows, past, Hq, H, D, P, qt, ot, window=0, sinks=0, seed=1, holes=(), pad=0, max_rows=None,
             work="auto"):
    n = len(rows)
    lens = [a + b for a, b in zip(rows, past)]
    pages = R.Pages(kv, H, D, P, n, max(1, (max(lens) + P - 1) // P + 1), seed)
    for s, T in enumerate(lens):
        if T:
            pages.put(s, _normal(seed * 100 + s, T, H, D), _normal(seed * 100 + 50 + s, T, H, D))
    for s, p in holes:
        pages.table[s, p] = -1
    cache = pages.cache(bq)
    total = sum(rows)
    q = (_normal(seed + 7, total, Hq * D) * 2).to(DT[qt])
    gq = torch.full((total, Hq * D + pad), float("nan"), dtype=DT[qt], device="cuda")
    gq[:, : Hq * D] = q.cuda()
    out = torch.full((total, Hq * D + pad), float("nan"), dtype=DT[ot], device="cuda")
    row0 = torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32, device="cuda")
    bq.Attention(cache, gq[:, : Hq * D], out[:, : Hq * D], torch.tensor(lens, dtype=torch.int32, device="cuda"),
                 window=window, sinks=sinks, row0=row0, max_rows=max_rows or max(rows), work=work).prefill()
    torch.cuda.synchronize()
    if pad:
        assert torch.isnan(out[:, Hq * D:]).all()
    got = out[:, : Hq * D].cpu().double().reshape(total, Hq, D)
    qr = q.float().reshape(total, Hq, D)
    qr = R.bf16(qr).double() if kv == "bf16" else R.half_rows(qr)
    first = 0
    for s, (r, T) in enumerate(zip(rows, lens)):
        hidden = torch.zeros(T, dtype=torch.bool)
        for hs, p in holes:
            if hs == s:
                hidden[p * P:(p + 1) * P] = True
        if r:
            k, v = pages.kh[s], R.bf16(pages.v[s]).double()
            ref = R.attention(qr[first: first + r], k, v, torch.arange(T - r, T), D ** -0.5, window, sinks, hidden)
            _check(got[first: first + r], *ref, False, f"prefill seq {s}: {r} rows of {T} tokens")
        first += r


@pytest.mark.parametrize("kv", ["bf16", "q8"])
@pytest.mark.parametrize("D,Hq,H,P", [(64, 8, 8, 16), (128, 32, 4, 64), (128, 6, 2, 16), (256, 7, 1, 32), (256, 2, 2, 256)])
def test_prefill_ragged(bq, kv, D, Hq, H, P):
    _prefill(bq, kv, [1, 37, 0, 130, 64], [0, 5, 100, 200, 64], Hq, H, D, P, "bf16", "bf16", seed=D + Hq)


@pytest.mark.parametrize("kv", ["bf16", "q8"])
@pytest.mark.parametrize("qt,ot", [("f32", "bf16"), ("bf16", "f32"), ("f32", "f32")])
def test_prefill_types_and_strides(bq, kv, qt, ot):
    for D in (64, 128, 256):
        _prefill(bq, kv, [70, 9], [3, 0], 8, 2, D, 32, qt, ot, seed=D, pad=8)


@pytest.mark.parametrize("kv", ["bf16", "q8"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (64, 4), (100, 65), (128, 0)])
def test_prefill_window_and_sinks(bq, kv, window, sinks):
    _prefill(bq, kv, [150, 33], [300, 0], 8, 2, 128, 16, "bf16", "bf16", window, sinks, seed=window)
    _prefill(bq, kv, [40], [200], 3, 1, 64, 128, "f32", "bf16", window, sinks, seed=window + 1)


def test_prefill_unmapped_pages_and_wide_bound(bq):
    _prefill(bq, "bf16", [60, 20], [100, 12], 8, 2, 128, 16, "bf16", "bf16", seed=6, holes=[(0, 0), (0, 6), (1, 0), (1, 1)])
    _prefill(bq, "q8", [60, 20], [100, 12], 8, 2, 64, 64, "bf16", "bf16", seed=6, holes=[(0, 1)], max_rows=400)


@pytest.mark.parametrize("kv", ["bf16", "q8"])
@pytest.mark.parametrize("D,Hq,H,P", [(64, 4, 4, 16), (128, 8, 2, 64), (256, 6, 2, 32)])
def test_prefill_split(bq, kv, D, Hq, H, P):
    """Few rows over many tokens: pieces and their join, without a workspace, and with room for two pieces."""
    for work in ("auto", None, torch.empty(2 * 50 * Hq * (D + 2) + 9, device="cuda")):
        _prefill(bq, kv, [40, 0, 9, 1], [1500, 3, 700, 0], Hq, H, D, P, "bf16", "bf16", seed=D, work=work)
    _prefill(bq, kv, [33], [2100], Hq, H, D, P, "f32", "f32", 1300, 70, seed=D + 1)
    _prefill(bq, kv, [33, 12], [1900, 800], Hq, H, D, P, "bf16", "bf16", seed=D + 2, holes=[(0, 0), (0, 9), (1, 4)])


@pytest.mark.parametrize("D,Hq,H,P", [(64, 8, 1, 16), (128, 16, 2, 64), (256, 8, 1, 32), (128, 8, 1, 256)])
def test_prefill_many_rows_over_q8(bq, D, Hq, H, P):
    """Enough rows for the q8 tiles to be converted ahead; without the workspace they are converted on the way."""
    for work in ("auto", None):
        _prefill(bq, "q8", [260, 5, 0], [100, 400, 7], Hq, H, D, P, "bf16", "bf16", seed=D, work=work)
    _prefill(bq, "q8", [270], [150], Hq, H, D, P, "f32", "f32", 90, 20, seed=D + 1)
    _prefill(bq, "q8", [256, 40], [130, 60], Hq, H, D, P, "bf16", "bf16", seed=D + 2, holes=[(0, 0), (1, 0)])


def test_prefill_one_sequence_without_row0(bq):
    pages = R.Pages("bf16", 2, 128, 64, 1, 3, 2)
    pages.put(0, _normal(1, 150, 2, 128), _normal(2, 150, 2, 128))
    q = R.bf16(_normal(3, 50, 4 * 128))
    out = torch.empty((50, 4 * 128), device="cuda")
    bq.Attention(pages.cache(bq), q.cuda(), out, torch.tensor([150], dtype=torch.int32, device="cuda")).prefill()
    ref = R.attention(q.double().reshape(50, 4, 128), pages.k[0], pages.v[0], torch.arange(100, 150), 128 ** -0.5)
    _check(out.cpu().double().reshape(50, 4, 128), *ref, False, "prefill")


def test_runs_agree_bit_for_bit(bq):
    a = _decode(bq, "bf16", [3000, 100], 1, 8, 2, 128, 64, "f32", "f32", seed=11)
    for _ in range(3):
        assert torch.equal(a, _decode(bq, "bf16", [3000, 100], 1, 8, 2, 128, 64, "f32", "f32", seed=11))


def test_offsets_past_32_bits(bq):
    """A cache of more than 4 GiB: the same sequence through low and high pages."""
    H, D, P = 8, 256, 256
    page = bq.kv_page_bytes("bf16", H, D, P)
    n = (5 << 30) // page
    pages = torch.zeros((n, page), dtype=torch.uint8, device="cuda")
    T = 600
    k, v = (_normal(s, T, H * D).cuda() for s in (1, 2))
    q = _normal(3, 1, H * D).cuda()
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    outs = []
    for ids in ([0, 1, 2], [n - 1, n - 2, n - 3]):
        cache = bq.KvCache(pages, torch.tensor([ids], dtype=torch.int32, device="cuda"), "bf16", H, D, P)
        bq.Append(cache, torch.zeros((T, H * D), device="cuda"), k, v, pos, torch.empty((T, H * D), device="cuda")).run()
        o = torch.empty((1, H * D), device="cuda")
        bq.Attention(cache, q, o, torch.tensor([T], dtype=torch.int32, device="cuda")).decode()
        p = torch.empty((T, H * D), dtype=torch.bfloat16, device="cuda")
        bq.Attention(cache, k, p, torch.tensor([T], dtype=torch.int32, device="cuda")).prefill()
        outs.append((o, p))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    assert torch.isfinite(outs[0][0]).all() and (outs[0][0] != 0).any()


def test_refusals(bq):
    L = bq.load()
    H, D, P = 2, 128, 64
    pages = R.Pages("bf16", H, D, P, 2, 2, 6)
    cache = pages.cache(bq)
    q = torch.zeros((2, 4 * D + 8), device="cuda")
    out = torch.full((2, 4 * D), 7.0, device="cuda")
    lens = torch.tensor([1, 1], dtype=torch.int32, device="cuda")
    ok = bq.Attention(cache, q[:, : 4 * D], out, lens)

    def call(f, kv=None, **change):
        a, c = bq.AttnArgs.from_buffer_copy(ok.struct), bq.KvCacheStruct.from_buffer_copy(cache.struct)
        for k, v in change.items():
            setattr(a, k, v)
        for k, v in (kv or {}).items():
            setattr(c, k, v)
        return f(ctypes.byref(c), ctypes.byref(a), bq._stream())

    E, U = bq.BQ_EINVAL, bq.BQ_UNSUPPORTED
    row0 = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    for f, extra in ((L.bq_attn_decode, {}), (L.bq_attn_prefill, dict(row0=row0.data_ptr()))):
        for change in (dict(q=None), dict(out=None), dict(kv_len=None), dict(q=q.data_ptr() + 4), dict(q_type=8),
                       dict(out_type=13), dict(q_heads=0), dict(rows=0), dict(max_len=-1), dict(window=-1), dict(sinks=-1),
                       dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=-1.0),
                       dict(ldq=4 * D - 8), dict(ldq=4 * D + 4), dict(ldo=0)):
            assert call(f, **{**extra, **change}) == E, (f, change)
        assert call(f, **{**extra, "q_heads": 3}) == U
        assert call(f, dict(head_dim=80), **extra) == U
        assert call(f, dict(table=None), **extra) == E
    assert call(L.bq_attn_decode, n_rows=3) == E
    assert call(L.bq_attn_decode, row0=row0.data_ptr()) == E
    assert call(L.bq_attn_decode, rows=9, n_rows=18) == U
    assert call(L.bq_attn_decode, work=None, work_bytes=4) == E
    assert call(L.bq_attn_prefill) == E  # two sequences without row0
    torch.cuda.synchronize()
    assert (out == 7).all()
    with pytest.raises(ValueError):
        bq.Attention(cache, q[:, : 4 * D], out, lens.long())
    with pytest.raises(TypeError):
        bq.Attention(cache, q[:, : 4 * D].half(), out, lens)


@pytest.mark.parametrize("powers", [(0, 0, 0, 0), (-30, -30, -30, -30), (12, 12, 12, 12), (0, 14, -25, 3), (40, 10, -10, -40)])
def test_prefill_many_rows_over_q8_value_ranges(bq, powers):
    """Values of every size, 64 tokens to a power of two: converted tiles keep fp32's range, and their products
    with the weights are fp16's where they are bf16's otherwise."""
    D, Hq, H, P, T = 128, 16, 2, 32, 256
    pages = R.Pages("q8", H, D, P, 1, T // P, 3)
    k, v = _normal(41, T, H, D), _normal(42, T, H, D)
    for i, p in enumerate(powers):
        v[64 * i: 64 * (i + 1)] *= 2.0 ** p
    pages.put(0, k, v)
    q = _normal(43, T, Hq * D) * 2
    out = torch.empty((T, Hq * D), device="cuda")
    att = bq.Attention(pages.cache(bq), q.cuda(), out, torch.tensor([T], dtype=torch.int32, device="cuda"))
    assert att.struct.work_bytes > 0
    att.prefill()
    got = out.cpu().double().reshape(T, Hq, D)
    ref, bound, A = R.attention(R.half_rows(q.reshape(T, Hq, D)), pages.kh[0], pages.v[0], torch.arange(T), D ** -0.5)
    # a value's and a weight's rounding to fp16: 2^-11 of a term each at most, or 2^-25 of the tile's range
    # (values up to 2^16, weights up to 2^15); fp32 sums as in the other tests
    tol = 2.0 ** -9 + 2.0 ** -18 * A[..., None]
    ratio = ((got - ref).abs() / (tol * bound).clamp(min=1e-300)).max().item()
    print(f"  {powers}: worst error / tolerance {ratio:.3f}", flush=True)
    assert ratio <= 1

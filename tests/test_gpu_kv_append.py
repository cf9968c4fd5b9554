"""bq_append and bq_kv_read against the 64-bit reference (tests/serve_ref.py).

Tolerances.  An fp32 query or key value is a few fp32 operations on values of
the head: |error| <= 2^-20 of the rotated pair's length (norm: a sum of D
squares, a root, two products; rotation: two products and a sum), and a bf16
one that plus half a bf16 step (8 significant bits: 2^-8 of the value).  A value passes unchanged:
bf16 pages are the rounded input bit for bit.  q8: the stored scale is
bf16(amax / 127), a step of at most amax / 127 (1 + 2^-8); the value is within
half a step (plus the fp32 error), or within amax - 127 scale where the scale
was rounded down, which is less.
"""
import ctypes

import numpy as np
import pytest
import torch

import serve_ref as R

pytestmark = pytest.mark.gpu


def _rows(seed, rows, width):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal((rows, width)).astype(np.float32) * 2)


def _inputs(rows, Hq, H, D, rot, n_pos, seed, norm):
    qkv = _rows(seed, rows, (Hq + 2 * H) * D)
    cs = torch.from_numpy(np.random.default_rng(seed + 1).uniform(-np.pi, np.pi, (n_pos, rot // 2))) if rot else None
    rope = torch.cat([cs.cos(), cs.sin()], 1).float() if rot else None
    w = [1 + 0.3 * _rows(seed + 2 + i, 1, D)[0] for i in range(2)] if norm else [None, None]
    return qkv, rope, w


def _reference(qkv, pos, rope, rot, w, Hq, H, D, inter, eps):
    x = qkv.double()
    q, k, v = (t.reshape(len(x), -1, D) for t in (x[:, : Hq * D], x[:, Hq * D:(Hq + H) * D], x[:, (Hq + H) * D:]))
    return R.append(q, k, v, pos.long(), None if rope is None else rope.double(), rot,
                    *(None if t is None else t.double() for t in w), eps, inter)


def _bound(ref, rot, inter):
    """2^-20 of the rotated pair's length, per value."""
    a = ref.abs().clone()
    for i in range(rot // 2):
        j, l = (2 * i, 2 * i + 1) if inter else (i, i + rot // 2)
        n = torch.hypot(ref[..., j], ref[..., l])
        a[..., j], a[..., l] = n, n
    return a * 2.0 ** -20 + 1e-30


CASES = [  # rows, n_seq, first positions' kind, Hq, H, D, P, rot, interleaved, norm
    (1, 1, "one", 32, 4, 128, 64, 128, False, True),
    (7, 7, "one", 8, 2, 128, 16, 64, True, True),
    (100, 1, "run", 16, 4, 128, 32, 128, False, False),
    (133, 3, "run", 6, 2, 64, 16, 32, False, True),
    (50, 2, "run", 4, 4, 256, 128, 256, True, True),
    (40, 2, "mixed", 3, 1, 64, 64, 8, False, True),
    (17, 1, "run", 7, 1, 256, 256, 0, False, False),
]


@pytest.mark.parametrize("kv", ["bf16", "q8"])
@pytest.mark.parametrize("rows,n_seq,kind,Hq,H,D,P,rot,inter,norm", CASES)
def test_append_matches_reference(bq, kv, rows, n_seq, kind, Hq, H, D, P, rot, inter, norm):
    print(f"append {kv} rows {rows} D {D} P {P}", flush=True)
    seed = rows * 7 + D
    n_pos = 640
    qkv, rope, w = _inputs(rows, Hq, H, D, rot, n_pos, seed, norm)
    rng = np.random.default_rng(seed + 9)
    seq = np.sort(rng.integers(0, n_seq, rows)) if kind != "one" else np.arange(rows)
    start = rng.integers(0, 300, n_seq)
    pos = np.array([start[s] + int((seq[:i] == s).sum()) for i, s in enumerate(seq)], np.int32)
    if kind == "mixed":  # rows in any order, padding rows and a position past the table's
        perm = rng.permutation(rows)
        seq, pos = seq[perm], pos[perm]
        pos[3], pos[11] = -1, n_pos
    pages = R.Pages(kv, H, D, P, n_seq, (n_pos + P - 1) // P, seed)
    cache = pages.cache(bq)
    before = cache.pages.clone()
    g, gp, gs = qkv.cuda(), torch.from_numpy(pos).cuda(), torch.from_numpy(seq.astype(np.int32)).cuda()
    cut = (Hq * D, (Hq + H) * D)
    gw = [None if t is None else t.cuda() for t in w]
    outs = {}
    for dt in (torch.float32, torch.bfloat16):
        cache.pages.copy_(before)
        q_out = torch.full((rows, Hq * D), float("nan"), dtype=dt, device="cuda")
        bq.Append(cache, g[:, : cut[0]], g[:, cut[0]: cut[1]], g[:, cut[1]:], gp, q_out, seq=gs, q_weight=gw[0],
                  k_weight=gw[1], eps=1e-5, rope=None if rope is None else rope.cuda(), n_pos=n_pos,
                  interleaved=inter).run()
        outs[dt] = q_out
    live = torch.from_numpy((pos >= 0) & (pos < n_pos))
    rq, rk, rv = _reference(qkv, torch.from_numpy(np.where(live, pos, 0)), rope, rot, w, Hq, H, D, inter, 1e-5)
    rq[~live] = 0
    tq = _bound(rq, rot, inter)
    for dt, half in ((torch.float32, 0.0), (torch.bfloat16, 2.0 ** -8)):
        err = (outs[dt].cpu().double().reshape(rq.shape) - rq).abs()
        assert (err <= tq + half * rq.abs()).all(), (dt, (err / (tq + half * rq.abs())).max())
    # the cache, through the address formulas
    raw = cache.pages.cpu().reshape(pages.n_pages, H, -1)
    t, h, d = torch.from_numpy(pos % P).long()[:, None, None], torch.arange(H)[None, :, None], torch.arange(D)[None, None]
    page = pages.table[torch.from_numpy(seq).long(), torch.from_numpy(np.where(live, pos, 0) // P).long()].long()[:, None, None]
    want = before.cpu().reshape(raw.shape).clone()
    got = {}
    for value, ref, r_ in ((0, rk, rot), (1, rv, 0)):
        if kv == "bf16":
            at = R.addr_bf16(P, D, t, d, value)
            x = raw.view(torch.bfloat16)[page, h, at]
            want.view(torch.bfloat16)[page[live], h, at[live]] = x[live]
            step = 2.0 ** -8 * ref.abs()
            if value:
                assert torch.equal(x[live].float(), R.bf16(ref)[live].float())
        else:
            code, sc = R.addr_q8(P, D, t, d, value)
            c, s = raw.view(torch.int8)[page, h, code], raw.view(torch.bfloat16)[page, h, sc // 2]
            want.view(torch.int8)[page[live], h, code[live]] = c[live]
            want.view(torch.bfloat16)[page[live], h, sc[live] // 2] = s[live]
            amax = ref.reshape(rows, H, -1, 32).abs().amax(-1).repeat_interleave(32, -1)
            assert ((s.double() - amax / 127).abs() <= (2.0 ** -8 + 2.0 ** -18) * amax / 127)[live].all()
            assert (c[live].int().abs() <= 127).all()
            x = c.double() * s.double()
            step = amax / 127 * (1 + 2.0 ** -8) / 2
        got[value] = x
        err = (x.double() - ref).abs()[live]
        tol = (_bound(ref, r_, inter) * 4 + step)[live]
        assert (err <= tol).all(), (value, (err / tol).max())
    assert torch.equal(raw, want), "bytes of other tokens changed"
    # read back: the same values as bf16, zeros for padding
    ko, vo = (torch.full((rows, H * D), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    cache.read(gp, ko, vo, seq=gs)
    for o, x in ((ko, got[0]), (vo, got[1])):
        ref = torch.where(live[:, None, None], R.bf16(x.float()), torch.zeros((), dtype=torch.bfloat16))
        inside = live.clone()
        inside[torch.from_numpy(pos < 0)] = True  # (a position past n_pos may still be mapped)
        assert torch.equal(o.cpu().reshape(ref.shape)[inside].float(), ref[inside].float())


def test_append_leaves_unmapped_pages_and_foreign_sequences(bq):
    H, D, P = 2, 64, 16
    pages = R.Pages("bf16", H, D, P, 2, 4, 5)
    pages.table[0, 1], pages.table[1, 0] = -1, pages.n_pages
    cache = pages.cache(bq)
    before = cache.pages.clone()
    rows = 6
    g = _rows(3, rows, 3 * H * D).cuda()
    pos = torch.tensor([16, 20, 3, 64, 5, 5], dtype=torch.int32, device="cuda")  # unmapped, unmapped, out of range page, past the table
    seq = torch.tensor([0, 0, 1, 0, 2, -1], dtype=torch.int32, device="cuda")    # ..., no such sequences
    q_out = torch.zeros((rows, H * D), device="cuda")
    bq.Append(cache, g[:, : H * D], g[:, H * D: 2 * H * D], g[:, 2 * H * D:], pos, q_out, seq=seq).run()
    assert torch.equal(cache.pages, before)
    want = g[:, : H * D].clone()
    want[4:] = 0
    assert torch.equal(q_out, want)
    k = torch.full((rows, H * D), float("nan"), dtype=torch.bfloat16, device="cuda")
    cache.read(pos, k=k, seq=seq)
    assert (k == 0).all()


def test_queries_in_place_and_on_another_stream(bq):
    H, D, P, rows = 2, 128, 64, 9
    cache = R.Pages("bf16", H, D, P, 1, 4, 6).cache(bq)
    g = _rows(8, rows, 8 * D).cuda()
    kvr = _rows(9, rows, 2 * H * D).cuda()
    rope = bq.rope_table(256, D)
    pos = torch.arange(100, 100 + rows, dtype=torch.int32, device="cuda")
    sep = torch.zeros_like(g)
    bq.Append(cache, g, kvr[:, : H * D], kvr[:, H * D:], pos, sep, rope=rope).run()
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        bq.Append(cache, g, kvr[:, : H * D], kvr[:, H * D:], pos, g, rope=rope).run()
    st.synchronize()
    assert torch.equal(sep, g)


def test_refusals(bq):
    L = bq.load()
    H, D, P, rows = 2, 128, 64, 4
    pages = R.Pages("bf16", H, D, P, 1, 2, 6)
    cache = pages.cache(bq)
    g = torch.zeros((rows, 8 * D + 4), device="cuda")
    pos = torch.arange(rows, dtype=torch.int32, device="cuda")
    q_out = torch.full((rows, 4 * D), 7.0, device="cuda")
    ok = bq.Append(cache, g[:, : 4 * D], g[:, 4 * D: 6 * D], g[:, 6 * D: 8 * D], pos, q_out, rope=bq.rope_table(8, D))

    def call(kv=None, **change):
        a, c = bq.AppendArgs.from_buffer_copy(ok.struct), bq.KvCacheStruct.from_buffer_copy(cache.struct)
        for k, v in change.items():
            setattr(a, k, v)
        for k, v in (kv or {}).items():
            setattr(c, k, v)
        return L.bq_append(ctypes.byref(c), ctypes.byref(a), bq._stream())

    E, U = bq.BQ_EINVAL, bq.BQ_UNSUPPORTED
    for change in (dict(q=None), dict(k=None), dict(v=None), dict(pos=None), dict(q_out=None), dict(rows=-1), dict(q_heads=0),
                   dict(q=g.data_ptr() + 4), dict(k_weight=g.data_ptr() + 4), dict(ldq=4 * D - 4), dict(ldk=8 * D + 2),
                   dict(rot=12), dict(rot=D + 8), dict(rope=None), dict(q_type=8), dict(n_pos=-1),
                   dict(q_out=g.data_ptr())):
        assert call(**change) == E, change
    for kv in (dict(pages=None), dict(table=None), dict(n_pages=0), dict(max_pages=0), dict(n_seq=0),
               dict(pages=cache.pages.data_ptr() + 8)):
        assert call(kv) == E, kv
    for kv in (dict(head_dim=96), dict(page_tokens=48), dict(page_tokens=8), dict(type=13), dict(max_pages=1 << 26)):
        assert call(kv) == U, kv
    assert call(rows=0) == bq.BQ_OK
    assert L.bq_kv_page_bytes(30, 4, 96, 64) == 0 and L.bq_kv_page_bytes(30, 4, 128, 64) == 4 * 4 * 64 * 128
    assert L.bq_kv_page_bytes(8, 4, 128, 64) == 4 * (2 * 64 * 128 + 64 * 128 // 8)
    torch.cuda.synchronize()
    assert (q_out == 7).all()
    with pytest.raises(ValueError):
        bq.Append(cache, g[:, : 4 * D], g[:, 4 * D: 6 * D], g[:, 6 * D: 8 * D], pos.long(), q_out)
    with pytest.raises(ValueError):
        bq.Append(cache, g[:3, : 4 * D], g[:, 4 * D: 6 * D], g[:, 6 * D: 8 * D], pos, q_out)

"""bq_append of long prompts, and of rows whose values are not numbers or very small
(reference and tolerances: test_gpu_kv_append.py)."""
import pytest
import torch

import serve_ref as R
from test_gpu_kv_append import _rows, test_append_matches_reference as _matches

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["bf16", "q8"])
@pytest.mark.parametrize("rows,n_seq,kind,Hq,H,D,P,rot,inter,norm", [
    (1025, 4, "run", 3, 2, 64, 16, 64, False, True),
    (1100, 5, "run", 5, 1, 128, 64, 128, False, True),
    (1030, 4, "run", 2, 2, 256, 128, 128, True, False),
    (1040, 5, "mixed", 2, 1, 128, 32, 64, False, True),
])
def test_prompts_match_reference(bq, kv, rows, n_seq, kind, Hq, H, D, P, rot, inter, norm):
    """Past 1024 rows a workgroup takes 16 rows of a head and stores 8 neighbouring tokens of a value as one unit."""
    _matches(bq, kv, rows, n_seq, kind, Hq, H, D, P, rot, inter, norm)


@pytest.mark.parametrize("kv", ["bf16", "q8"])
@pytest.mark.parametrize("D,P", [(64, 16), (128, 64), (256, 256)])
def test_prompt_equals_its_pieces(bq, kv, D, P):
    """A prompt in one call and in calls of a few rows gives the same pages and queries, bit for bit."""
    H, Hq, rows, at = 2, 4, 1500, 5
    g = _rows(D, rows, (Hq + 2 * H) * D).cuda()
    pos = torch.arange(at, at + rows, dtype=torch.int32, device="cuda")
    rope = bq.rope_table(at + rows, D)
    table = torch.arange((at + rows + P - 1) // P, dtype=torch.int32, device="cuda").flip(0)[None].contiguous()
    cut, made = (Hq * D, (Hq + H) * D), []
    for step in (rows, 700, 33):
        cache = bq.KvCache.empty(table.shape[1], table, kv, H, D, P)
        q = torch.empty((rows, Hq * D), device="cuda")
        for a in range(0, rows, step):
            x = g[a: a + step]
            bq.Append(cache, x[:, : cut[0]], x[:, cut[0]: cut[1]], x[:, cut[1]:], pos[a: a + step], q[a: a + step], rope=rope).run()
        made.append((cache.pages, q))
    for pages, q in made[1:]:
        assert torch.equal(pages, made[0][0]) and torch.equal(q, made[0][1])


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


@pytest.mark.parametrize("rows", [12, 1100])
@pytest.mark.parametrize("size", [1e-30, 1e-35, 1e-36, 1e-37, 4e-38])
def test_codes_of_tiny_values(bq, rows, size):
    """Codes are taken against the stored scale where its reciprocal passes fp32's range, too."""
    H, D, P = 1, 64, 32
    k, v = (_rows(s, rows, D) * size for s in (5, 6))
    cache, _ = _append_raw(bq, "q8", k, v, P)
    raw = cache.pages.cpu().reshape(cache.pages.shape[0], H, -1)
    t, d = torch.arange(rows)[:, None], torch.arange(D)[None]
    page = cache.table.cpu()[0][torch.arange(rows) // P].long()[:, None]
    for value, x in ((0, k), (1, v)):
        code, sc = R.addr_q8(P, D, t % P, d, value)
        c = raw.view(torch.int8)[page, 0, code].double()
        s = raw.view(torch.bfloat16)[page, 0, sc // 2].double()
        amax = x.double().reshape(rows, -1, 32).abs().amax(-1).repeat_interleave(32, -1)
        # bf16: half a step of 8 bits, or of 2^-133
        assert ((s - amax / 127).abs() <= torch.clamp(2.0 ** -8 * amax / 127, min=2.0 ** -134) * (1 + 2.0 ** -10)).all()
        want = torch.where(s > 0, (x.double() / s.clamp(min=2.0 ** -140)), torch.zeros(())).clamp(-127, 127)
        assert ((c - want).abs() <= 0.5 + 2.0 ** -10).all(), (size, (c - want).abs().max())

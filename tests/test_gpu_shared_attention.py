"""bq_attn_decode_shared against 64-bit attention over what the cache stands for
(tests/serve_ref.py).  A sequence's pages hold NaN (or are unmapped) where its group's
prefix would lie, and so does every other byte that holds no token, so a token read
through the wrong row of the table would show.

Tolerances as in test_gpu_attention.py, relative to sum_j p_j |v_j|: fp32 2^-16 + 2^-18 A,
bf16 weights and outputs 2^-7 (1 + 2^-6) + 2^-18 A.  The join adds a few fp32 roundings
(2^-24 each) to both.
"""
import ctypes

import numpy as np
import pytest
import torch

import serve_ref as R
from test_gpu_attention import DT, _check, _normal

pytestmark = pytest.mark.gpu
NAN = float("nan")


class Batch:
    """Sequences in groups over one cache.  groups: (sequences, shared tokens) of each, own: tokens of each sequence
    behind the prefix (negative: shorter than it), the sequences behind the last group have none."""

    def __init__(self, kv, H, D, P, groups, own, seed, holes=(), lead=0):
        self.n, self.P = len(own), P
        self.group0 = [lead + sum(g[0] for g in groups[:i]) for i in range(len(groups) + 1)]
        self.prefix = [g[1] for g in groups]
        of = lambda s: next((g for g in range(len(groups)) if self.group0[g] <= s < self.group0[g + 1]), -1)
        self.group = [of(s) for s in range(self.n)]
        shared = [self.prefix[g] if g >= 0 else 0 for g in self.group]
        self.lens = [max(0, c + o) for c, o in zip(shared, own)]
        # a first sequence that is shorter than its prefix still has all of it in the cache
        hold = [max(T, c) if self.group0[max(g, 0)] == s and g >= 0 else T
                for s, (T, c, g) in enumerate(zip(self.lens, shared, self.group))]
        pages = self.pages = R.Pages(kv, H, D, P, self.n, max(1, (max(hold) + P - 1) // P + 1), seed)
        for s, g in enumerate(self.group):
            k, v = _normal(seed * 100 + s, hold[s], H, D), _normal(seed * 100 + 50 + s, hold[s], H, D)
            if g >= 0 and s != self.group0[g]:
                k[: shared[s]], v[: shared[s]] = NAN, NAN
            if hold[s]:
                pages.put(s, k, v)
            if g >= 0 and s != self.group0[g]:
                pages.table[s, : shared[s] // P] = -1 if s % 2 else pages.table[s, 0]
        for s, p in holes:
            pages.table[s, p] = -1
        self.holes = holes

    def tokens(self, s):
        """K, V and the unmapped tokens of sequence s, the prefix from the group's first."""
        T, g = self.lens[s], self.group[s]
        if T == 0:
            return None
        if g < 0 or s == self.group0[g]:
            k, v, c, first = self.pages.k[s][:T], self.pages.v[s][:T], 0, s
        else:
            c, first = min(self.prefix[g], T), self.group0[g]
            k = torch.cat([self.pages.k[first][:c], self.pages.k[s][c:T]])
            v = torch.cat([self.pages.v[first][:c], self.pages.v[s][c:T]])
        at = torch.arange(T) // self.P
        hidden = torch.zeros(T, dtype=torch.bool)
        for hs, p in self.holes:
            if hs == first:
                hidden |= (at == p) & (torch.arange(T) < c)
            if hs == s:
                hidden |= (at == p) & (torch.arange(T) >= c)
        return k, v, hidden


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _buffers(b, rows, Hq, D, qt, ot, seed, pad, qscale):
    q = (_normal(seed + 7, b.n * rows, Hq * D) * qscale).to(DT[qt])
    gq = torch.full((b.n * rows, Hq * D + pad), NAN, dtype=DT[qt], device="cuda")
    gq[:, : Hq * D] = q.cuda()
    return q, gq, torch.full((b.n * rows, Hq * D + pad), NAN, dtype=DT[ot], device="cuda")


def _verify(b, out, q, rows, Hq, H, D, fine, window=0, sinks=0, what=""):
    got = out.cpu().double().reshape(b.n, rows, Hq, D)
    for s, T in enumerate(b.lens):
        if T:
            k, v, hidden = b.tokens(s)
            ref = R.attention(q[s * rows:(s + 1) * rows].double().reshape(rows, Hq, D), k, v, torch.arange(T - rows, T), D ** -0.5,
                              window, sinks, hidden)
        else:
            ref = [torch.zeros((rows, Hq, D), dtype=torch.float64)] * 2 + [torch.zeros((rows, Hq), dtype=torch.float64)]
        _check(got[s], *ref, fine, f"{what} seq {s} of {T} tokens, group {b.group[s]}")


def _shared(bq, kv, groups, own, rows, Hq, H, D, P, qt, ot, window=0, sinks=0, seed=1, holes=(), pad=0, qscale=2.0, lead=0,
            max_len=None, max_prefix=None):
    b = Batch(kv, H, D, P, groups, own, seed, holes, lead)
    print(f"shared {kv} groups {groups} own {own} lead {lead} rows {rows} heads {Hq}/{H} D {D} P {P} {qt} {ot} window {window}/{sinks}",
          flush=True)
    q, gq, out = _buffers(b, rows, Hq, D, qt, ot, seed, pad, qscale)
    att = bq.SharedAttention(b.pages.cache(bq), gq[:, : Hq * D], out[:, : Hq * D], _ints(b.lens), _ints(b.group0), _ints(b.prefix),
                             window=window, sinks=sinks, max_len=max_len, max_prefix=max_prefix)
    att.work.fill_(NAN)
    att.run()
    torch.cuda.synchronize()
    if pad:
        assert torch.isnan(out[:, Hq * D:]).all()
    _verify(b, out[:, : Hq * D], q, rows, Hq, H, D, qt == "f32" and ot == "f32", window, sinks)
    return b, q, gq, out


@pytest.mark.parametrize("kv", ["bf16", "q8"])
@pytest.mark.parametrize("D,Hq,H,P", [(64, 8, 8, 16), (128, 32, 4, 64), (128, 6, 2, 16), (256, 7, 1, 32), (256, 2, 2, 256)])
def test_lengths(bq, kv, D, Hq, H, P):
    """Prefixes of one token, inside a page, of whole pages and none; own tokens from one on; sequences that are as
    long as the prefix, shorter, empty, or in no group."""
    _shared(bq, kv, [(3, 70), (2, 1), (1, 33), (2, 0), (4, 256)], [1, 5, 40, 3, 64, 2, 9, 31, 1, 0, -100, -256, 50, 0], 1, Hq, H, D, P,
            "f32", "f32", seed=D + Hq)


@pytest.mark.parametrize("kv", ["bf16", "q8"])
@pytest.mark.parametrize("qt,ot", [("f32", "bf16"), ("bf16", "f32"), ("bf16", "bf16")])
def test_types_and_strides(bq, kv, qt, ot):
    for D in (64, 128, 256):
        _shared(bq, kv, [(5, 100)], [3, 60, 1, 17, 33], 1, 8, 2, D, 32, qt, ot, seed=D, pad=8)


@pytest.mark.parametrize("kv", ["bf16", "q8"])
@pytest.mark.parametrize("rows", [2, 5, 8])
def test_verify_rows(bq, kv, rows):
    """Several new tokens, some of whose positions lie in the prefix or before the first token."""
    _shared(bq, kv, [(4, 50), (2, 6)], [rows, 1, 0, 40, 2 - rows, rows], rows, 24, 2, 128, 16, "f32", "f32", seed=rows)
    _shared(bq, kv, [(2, 90)], [7, 30, 4], rows, 5, 5, 64, 64, "bf16", "bf16", seed=rows + 20)


@pytest.mark.parametrize("kv", ["bf16", "q8"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 3), (64, 0), (100, 33), (300, 90), (200, 260)])
def test_window_and_sinks(bq, kv, window, sinks):
    """Windows that end before, inside and behind the prefix, at another place for each sequence; sinks that reach
    past the prefix."""
    for rows, types in ((1, ("f32", "f32")), (6, ("bf16", "bf16"))):
        _shared(bq, kv, [(4, 150), (2, 45)], [9, 64, 210, 1, 300, 20], rows, 8, 2, 128, 16, *types, window, sinks, seed=window + rows)
    _shared(bq, kv, [(3, 333)], [400, 2, 61], 1, 8, 2, 64, 128, "f32", "f32", window, sinks, seed=window)


@pytest.mark.parametrize("kv", ["bf16", "q8"])
def test_unmapped_pages(bq, kv):
    """Of the prefix (through the first sequence's row) and of a sequence's own tokens."""
    _shared(bq, kv, [(3, 120)], [40, 70, 12, 33], 2, 8, 2, 128, 16, "f32", "f32", seed=6, holes=[(0, 2), (0, 7), (1, 8), (3, 0)])
    _shared(bq, kv, [(2, 128)], [1, 1], 1, 8, 2, 64, 64, "f32", "f32", seed=7, holes=[(0, 0), (0, 1)])


@pytest.mark.parametrize("kv", ["bf16", "q8"])
@pytest.mark.parametrize("D,Hq,H,P", [(64, 12, 3, 16), (128, 32, 4, 64), (256, 8, 1, 32)])
def test_long_prefixes(bq, kv, D, Hq, H, P):
    """Pieces of the prefix and of the own tokens, and their join; many rows a group."""
    for types in (("f32", "f32"), ("bf16", "bf16")):
        _shared(bq, kv, [(20, 3001)], [17 * i % 90 + 1 for i in range(20)], 1, Hq, H, D, P, *types, seed=D)
    _shared(bq, kv, [(2, 1500), (7, 700)], [1300, 3, 800, 1, 2, 40, 5, 77, 600], 3, Hq, H, D, P, "f32", "f32", 1000, 5, seed=D + 1)


@pytest.mark.parametrize("kv", ["bf16", "q8"])
@pytest.mark.parametrize("D,Hq,H", [(64, 64, 8), (128, 32, 4), (256, 24, 3)])
def test_rows_that_fill_the_chip(bq, kv, D, Hq, H):
    """Enough rows and tokens that two row tiles share a step, with a broken tile at the end of each group."""
    for rows, types, window, sinks in ((1, ("f32", "f32"), 0, 0), (2, ("bf16", "bf16"), 0, 0), (1, ("f32", "f32"), 1500, 40)):
        _shared(bq, kv, [(9, 2100), (2, 1900), (6, 800)], [1 + 7 * i % 40 for i in range(17)], rows, Hq, H, D, 64, *types, window, sinks,
                seed=D + rows)


def test_sequences_before_the_first_group(bq):
    _shared(bq, "bf16", [(3, 60)], [100, 33, 5, 6, 70, 2], 1, 8, 2, 128, 16, "f32", "f32", seed=11, lead=2)


@pytest.mark.parametrize("kv", ["bf16", "q8"])
def test_peaked_scores(bq, kv):
    """Scores tens apart: all the weight in the prefix for some rows, none for others."""
    _shared(bq, kv, [(9, 400)], list(range(20, 200, 20)), 1, 16, 2, 128, 32, "f32", "f32", seed=5, qscale=25.0)


def test_one_group_a_sequence(bq):
    """Groups of one: bq_attn_decode with its tokens cut in two; and many groups (more than a wave has lanes)."""
    _shared(bq, "bf16", [(1, 3 + 7 * i % 50) for i in range(70)], [1 + i % 9 for i in range(70)], 1, 4, 2, 64, 16, "f32", "f32", seed=12)
    _shared(bq, "q8", [(0, 9), (2, 40), (0, 77), (0, 1), (1, 20)], [5, 6, 7], 1, 4, 2, 64, 16, "f32", "f32", seed=13)


def test_lengths_are_clamped(bq):
    """max_len and max_prefix bound what the device memory says."""
    b = Batch("bf16", 2, 64, 16, [(2, 40)], [30, 8], 14)
    q, gq, out = _buffers(b, 1, 4, 64, "f32", "f32", 14, 0, 2.0)
    att = bq.SharedAttention(b.pages.cache(bq), gq, out, _ints([50, 48]), _ints(b.group0), _ints([4000]), max_len=50, max_prefix=40)
    att.run()
    b.lens = [50, 48]
    _verify(b, out, q, 1, 4, 2, 64, True)


@pytest.mark.parametrize("kv", ["bf16", "q8"])
def test_same_tokens_as_decode(bq, kv):
    """Pages that all rows of the table share: what bq_attn_decode gives, up to rounding."""
    n, prefix, P, H, Hq, D = 6, 64, 16, 2, 8, 128
    pages = R.Pages(kv, H, D, P, n, 8, 15)
    own = [3, 40, 17, 1, 64, 30]
    for s in range(n):
        pages.put(s, _normal(900 + s, prefix + own[s], H, D), _normal(950 + s, prefix + own[s], H, D))
    pages.table[1:, : prefix // P] = pages.table[0, : prefix // P]
    cache, lens = pages.cache(bq), _ints([prefix + o for o in own])
    q = _normal(16, n, Hq * D).cuda() * 2
    a, b = torch.full_like(q, NAN), torch.full_like(q, NAN)
    bq.Attention(cache, q, a, lens).decode()
    bq.SharedAttention(cache, q, b, lens, _ints([0, n]), _ints([prefix])).run()
    # each is off by 2^-16 + 2^-18 A of sum p |v| (A below 60, |v| below 6)
    assert (a - b).abs().max().item() <= 2 * (2.0 ** -16 + 60 * 2.0 ** -18) * 6


def test_captured_and_replayed(bq):
    """Lengths change between a graph's replays, with eager work and synchronizations between; equal calls give equal
    bits."""
    b = Batch("bf16", 2, 128, 16, [(4, 130)], [30, 31, 5, 90, 20], 17)
    q, gq, out = _buffers(b, 1, 8, 128, "f32", "f32", 17, 0, 2.0)
    lens, group0, prefix = _ints(b.lens), _ints(b.group0), _ints(b.prefix)
    cache = b.pages.cache(bq)
    att = bq.SharedAttention(cache, gq, out, lens, group0, prefix, max_len=300, max_prefix=200)
    att.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        att.run()
    eager = torch.full_like(out, NAN)
    again = bq.SharedAttention(cache, gq, eager, lens, group0, prefix, max_len=300, max_prefix=200)
    for step in range(5):
        own = [30 - step, 31, 5 - step, 90, 20]
        b.lens = [130 + o for o in own[:4]] + [own[4]]
        lens.copy_(_ints(b.lens))
        out.fill_(NAN)
        graph.replay()
        torch.cuda.synchronize()
        first = out.clone()
        att.work.fill_(NAN)
        graph.replay()
        again.run()
        torch.cuda.synchronize()
        assert torch.equal(first, out) and torch.equal(first, eager), step
        _verify(b, out, q, 1, 8, 2, 128, True, what=f"replay {step}")


def test_two_calls_on_two_streams(bq):
    """Each with a workspace of its own."""
    jobs = []
    for i in range(2):
        b = Batch("q8" if i else "bf16", 2, 64, 16, [(6, 500 + i)], [40, 3, 9, 77, 1, 20], 18 + i)
        q, gq, out = _buffers(b, 1, 8, 64, "f32", "f32", 18 + i, 0, 2.0)
        att = bq.SharedAttention(b.pages.cache(bq), gq, out, _ints(b.lens), _ints(b.group0), _ints(b.prefix))
        jobs.append((b, q, out, att, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(3):
        for *_, att, st in jobs:
            with torch.cuda.stream(st):
                att.run()
    torch.cuda.synchronize()
    for b, q, out, _, _ in jobs:
        _verify(b, out, q, 1, 8, 2, 64, True)


def test_offsets_past_32_bits(bq):
    """Pages more than 2^31 bytes into the pool."""
    H, D, P = 4, 256, 256
    size = bq.kv_page_bytes("bf16", H, D, P)
    n_pages = (1 << 32) // size + 40
    table = torch.tensor([[n_pages - 1, n_pages - 5, n_pages - 2], [0, 1, n_pages - 3]], dtype=torch.int32, device="cuda")
    cache = bq.KvCache.empty(n_pages, table, "bf16", H, D, P)
    k = torch.zeros((3, H, D // 8, P, 8), dtype=torch.bfloat16, device="cuda")
    v = torch.arange(3, device="cuda").to(torch.bfloat16)[:, None, None].expand(3, H, P * D)
    for i, page in enumerate((n_pages - 1, n_pages - 5, n_pages - 3)):
        cache.pages[page].view(torch.bfloat16).view(H, 2, P * D).copy_(torch.stack([k[i].reshape(H, -1), v[i]], 1))
    q = torch.ones((2, 8 * D), device="cuda")
    out = torch.full_like(q, NAN)
    bq.SharedAttention(cache, q, out, _ints([512, 768]), _ints([0, 2]), _ints([512])).run()
    # equal scores: the mean over pages of values 0, 1 (first sequence) and 0, 1, 2 (second); sums of 768 exact values
    assert (out[0] - 0.5).abs().max().item() <= 2.0 ** -16 and (out[1] - 1).abs().max().item() <= 2.0 ** -16


def test_refusals(bq):
    H, D, P, n = 2, 64, 16, 3
    table = torch.zeros((n, 4), dtype=torch.int32, device="cuda")
    cache = bq.KvCache.empty(4, table, "bf16", H, D, P)
    q = torch.zeros((n, 4 * D), device="cuda")
    out = torch.full_like(q, 7.0)
    att = bq.SharedAttention(cache, q, out, _ints([9] * n), _ints([0, n]), _ints([4]))
    L, call = bq.load(), lambda: bq.load().bq_attn_decode_shared(cache.ref, ctypes.byref(att.struct), ctypes.byref(att.prefix), None)

    def refused(code, obj, **fields):
        keep = {f: getattr(obj, f) for f in fields}
        for f, v in fields.items():
            setattr(obj, f, v)
        assert call() == code, (fields, call())
        for f, v in keep.items():
            setattr(obj, f, v)
    E, U = bq.BQ_EINVAL, bq.BQ_UNSUPPORTED
    for fields in (dict(group0=None), dict(len=None), dict(n_groups=0), dict(n_groups=-1), dict(max_len=-1)):
        refused(E, att.prefix, **fields)
    for fields in (dict(q=None), dict(out=None), dict(kv_len=None), dict(rows=2), dict(n_rows=2), dict(scale=0.0), dict(scale=NAN),
                   dict(window=-1), dict(sinks=-1), dict(max_len=-1), dict(ldq=4), dict(q_type=13), dict(work=None),
                   dict(work_bytes=att.struct.work_bytes - 4), dict(work=att.struct.work + 4), dict(row0=att.prefix.group0)):
        refused(E, att.struct, **fields)
    refused(U, att.struct, q_heads=3)
    refused(U, att.struct, rows=9, n_rows=27)
    big = bq.KvCacheStruct.from_buffer_copy(cache.struct)
    big.n_seq, big.kv_heads = 65535, 64
    wide = bq.AttnArgs.from_buffer_copy(att.struct)
    wide.rows, wide.n_rows, wide.q_heads, wide.ldq, wide.ldo = 8, 8 * 65535, 64, 64 * D, 64 * D
    assert L.bq_attn_decode_shared(ctypes.byref(big), ctypes.byref(wide), ctypes.byref(att.prefix), None) == U   # more rows than a grid has
    assert L.bq_attn_decode_shared(None, ctypes.byref(att.struct), ctypes.byref(att.prefix), None) == E
    assert L.bq_attn_decode_shared(cache.ref, None, ctypes.byref(att.prefix), None) == E
    assert L.bq_attn_decode_shared(cache.ref, ctypes.byref(att.struct), None, None) == E
    torch.cuda.synchronize()
    assert (out == 7.0).all()
    size = L.bq_attn_shared_workspace_bytes
    assert size(n, 1, 4, H, D, 64, 1, 4) == att.struct.work_bytes
    for bad in ((0, 1, 4, 2, 64, 64, 1, 4), (3, 9, 4, 2, 64, 64, 1, 4), (3, 1, 3, 2, 64, 64, 1, 4), (3, 1, 4, 2, 64, 64, 0, 4), (3, 1, 4, 2, 64, -1, 1, 4)):
        assert size(*bad) == 0, bad


def test_groups_that_are_not_groups(bq):
    """group0 and len of any numbers: no access outside the buffers, and sequences of no group are right."""
    b = Batch("bf16", 2, 64, 16, [(0, 0)], [40, 3, 61, 17], 21)
    q, gq, out = _buffers(b, 1, 8, 64, "f32", "f32", 21, 0, 2.0)
    cache = b.pages.cache(bq)
    for group0, lens in (([9, 3, -5], [100, -4]), ([-7, -3, 0], [1 << 30, 5]), ([4, 4, 1 << 30], [-(1 << 31), 7])):
        out.fill_(NAN)
        bq.SharedAttention(cache, gq, out, _ints(b.lens), _ints(group0), _ints(lens)).run()
        torch.cuda.synchronize()
        _verify(b, out, q, 1, 8, 2, 64, True, what=f"group0 {group0}")


def test_hook(bq):
    """The attention hook takes the shared form where a block has one, and refuses it beside prefill."""
    b = Batch("bf16", 2, 128, 16, [(3, 50)], [20, 7, 31], 22)
    q, gq, out = _buffers(b, 1, 8, 128, "f32", "f32", 22, 0, 2.0)
    att = bq.SharedAttention(b.pages.cache(bq), gq, out, _ints(b.lens), _ints(b.group0), _ints(b.prefix))
    block = bq.AttnBlock(ctypes.pointer(att.kv.struct), None, ctypes.pointer(att.struct), 0, ctypes.pointer(att.prefix))
    plan = bq.AttnPlanStruct(1, ctypes.pointer(block), 0)
    bq.load().bq_attn_hook(ctypes.byref(plan), 0, None)
    torch.cuda.synchronize()
    assert plan.status == bq.BQ_OK
    _verify(b, out, q, 1, 8, 2, 128, True)
    block.prefill = 1
    bq.load().bq_attn_hook(ctypes.byref(plan), 0, None)
    assert plan.status == bq.BQ_EINVAL

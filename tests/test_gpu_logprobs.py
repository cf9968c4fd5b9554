"""bq_logprobs against the definition in 64 bits; ranks and alternatives exactly.

Tolerance.  x = (logit - max) / T takes three or four roundings (the difference, the factor log2(e) / T, the
product; or the difference and the quotient): 2^-22 |x|.  A weight e^x is off by that and by exp2's 2^-22 at
most, a sum of positive terms by 2^-24 per addition on a path of 16 + 6 + 2 in a slice and 8 over the slices:
2^-19.  With r = sum e^x over all but the first token, S1 = sum e^x |x|, S2 = sum e^x x^2:
  d r  <= 2^-19 r + 2^-22 (r + S1) + n 2^-126
  d S1 <= 2^-19 S1 + 2^-22 (2 S1 + S2) + n 2^-119
(a weight below 2^-126 is 0, as v_exp_f32 gives no denormal: each of n tokens is off by at most that, and
e^x |x| there by 2^-126 times ln 2^126 < 2^7, as x e^x falls from x = -1 down)
  d log p <= 2^-22 |x| + d r / (1 + r) + 2^-22 log(1 + r)
  d H  <= d r / (1 + r) + 2^-22 log(1 + r) + (d S1 + S1 d r / (1 + r)) / (1 + r) + 2^-22 H
"""
import ctypes

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -22
INF = np.float32(np.inf)


def _reference(logits, token, T, top):
    z = np.where(np.isnan(logits), -np.inf, logits.astype(np.float64))
    order = np.lexsort((np.arange(len(z)), -z))
    best, m = order[0], z[order[0]]
    rank = len(z) if not 0 <= token < len(z) else int(np.nonzero(order == token)[0][0])
    tops = [int(i) for i in order[:top]] + [-1] * (top - len(z))
    if not T > 0 or not np.isfinite(m):
        lp = lambda i: (0.0 if i == best else -np.inf, 0.0)
        H = (0.0, 0.0)
    else:
        with np.errstate(over="ignore", invalid="ignore"):
            x = np.where(z == -np.inf, -np.inf, (z - m) / np.float64(T))
        live = x > -np.inf
        live[best] = False
        xs = x[live]
        w = np.exp(xs)
        r, s1, s2 = w.sum(), (w * -xs).sum(), (w * xs * xs).sum()
        n = len(z)
        dr, ds = 2.0 ** -19 * r + U * (r + s1) + n * 2.0 ** -126, 2.0 ** -19 * s1 + U * (2 * s1 + s2) + n * 2.0 ** -119
        log_z = np.log1p(r)
        d_z = dr / (1 + r) + U * log_z

        def lp(i):
            return (x[i] - log_z, U * abs(x[i]) + d_z) if x[i] > -np.inf else (-np.inf, 0.0)
        h = log_z + s1 / (1 + r)
        H = (h, d_z + (ds + s1 * dr / (1 + r)) / (1 + r) + U * h)
    return {"logprob": lp(token) if 0 <= token < len(z) else (-np.inf, 0.0), "rank": rank, "entropy": H, "top": tops,
            "tops": [lp(i) if i >= 0 else (-np.inf, 0.0) for i in tops]}


def _close(got, want, what):
    v, tol = want
    if v == -np.inf:
        assert got == -np.inf, (what, got)
    elif v < -3.4028235e38:
        # below fp32's lowest number (-2^128 + 2^104; from half a step of 2^104 below it on, rounding gives -inf)
        assert got <= -3.402e38, (what, got)
    else:
        # 1e-44: a result below fp32's smallest number may be 0
        assert abs(float(got) - v) <= tol + 1e-44, (what, float(got), v, tol)


class Call:
    def __init__(self, bq, logits, tokens, temp, top, ld=None, want=("logprob", "rank", "entropy", "top_tokens", "top_logprobs")):
        rows, vocab = logits.shape
        self.host = logits
        buf = np.full((rows, ld or vocab), 1e30, np.float32)  # what lies between rows is not read
        buf[:, :vocab] = logits
        self.dev = torch.from_numpy(buf).cuda()
        self.tokens, self.temp, self.top = np.asarray(tokens, np.int32), None if temp is None else np.broadcast_to(np.float32(temp), (rows,)).copy(), top
        f = lambda *s: torch.full(s, float("nan"), device="cuda")
        i = lambda *s: torch.full(s, -7, dtype=torch.int32, device="cuda")
        self.out = {"logprob": f(rows), "rank": i(rows), "entropy": f(rows)}
        if top:
            self.out.update(top_tokens=i(rows, top), top_logprobs=f(rows, top))
        self.out = {k: v for k, v in self.out.items() if k in want}
        given = torch.from_numpy(self.tokens).cuda() if "logprob" in want or "rank" in want else None
        self.op = bq.LogProbs(self.dev[:, :vocab], tokens=given, temperature=None if temp is None else torch.from_numpy(self.temp).cuda(), **self.out)
        self.op.work.fill_(0xFF)

    def run(self):
        self.op.run()
        torch.cuda.synchronize()
        return self.check()

    def check(self):
        got = {k: v.cpu().numpy() for k, v in self.out.items()}
        for r in range(len(self.host)):
            ref = _reference(self.host[r], int(self.tokens[r]), 1.0 if self.temp is None else float(self.temp[r]), self.top)
            if "rank" in got:
                assert got["rank"][r] == ref["rank"], (r, got["rank"][r], ref["rank"])
            for k in ("logprob", "entropy"):
                if k in got:
                    _close(got[k][r], ref[k], (r, k))
            if "top_tokens" in got:
                assert got["top_tokens"][r].tolist() == ref["top"], r
            if "top_logprobs" in got:
                for j, want in enumerate(ref["tops"]):
                    _close(got["top_logprobs"][r][j], want, (r, "top", j))
        return got


def _peaked(seed, rows, vocab):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, vocab)).astype(np.float32) * 1.5
    for r in range(rows):
        x[r, rng.choice(vocab, min(40, vocab), replace=False)] += rng.uniform(4, 12, min(40, vocab)).astype(np.float32)
    return x, rng


@pytest.mark.parametrize("vocab", [1, 3, 63, 255, 4095, 4096, 4097, 8196, 32000, 131072, 262148])
@pytest.mark.parametrize("top", [0, 1, 2, 5, 20, 64])
def test_vocabularies(bq, vocab, top):
    """One slice to many, rows at any alignment, more alternatives than tokens."""
    x, rng = _peaked(vocab + top, 5, vocab)
    tokens = [0, vocab - 1, int(x[2].argmax()), rng.integers(vocab), int(x[4].argmin())]
    print(f"logprobs vocab {vocab} top {top}", flush=True)
    Call(bq, x, tokens, None, top, ld=vocab + 3).run()
    Call(bq, x, tokens, rng.uniform(0.3, 2, 5), top, ld=vocab).run()


@pytest.mark.parametrize("top", [1, 2, 20, 33, 64])
@pytest.mark.parametrize("kind", ["equal", "levels", "half", "rising", "falling", "block", "ties"])
def test_flat_and_ordered_rows(bq, kind, top):
    """Rows whose alternatives are many or lie together: ties go to the lower index."""
    rng = np.random.default_rng(top)
    vocab = 30001
    x = {"equal": lambda: np.zeros((3, vocab)),
         "levels": lambda: rng.integers(0, 3, (3, vocab)),
         "half": lambda: np.round(rng.standard_normal((3, vocab)) * 4) / 4,
         "rising": lambda: np.tile(np.arange(vocab) / 1000, (3, 1)),
         "falling": lambda: -np.tile(np.arange(vocab) / 1000, (3, 1)),
         "block": lambda: np.where((np.arange(vocab) >= 9000) & (np.arange(vocab) < 9100), 5.0, 0.0) + rng.standard_normal((3, vocab)) * 0.1,
         "ties": lambda: np.where(np.arange(vocab) % 4096 == 77, 3.0, np.arange(vocab) % 7 * 0.1) * np.ones((3, 1))}[kind]().astype(np.float32)
    Call(bq, x, [0, 17000, vocab - 1], None, top).run()


@pytest.mark.parametrize("temp", [1e-3, 0.05, 0.999, 1.0, 7.0, 1e4, 3e38, np.inf, 1e-30, 1e-42, 0.0, -1.0, np.nan])
def test_temperatures(bq, temp):
    x, rng = _peaked(9, 4, 9000)
    x[1, ::3] = -np.inf
    x[2] *= 1e-4
    x[3, 100] = 3e38
    x[3, 200:300] = -3e38
    Call(bq, x, [1, 3, 8999, 250], temp, 5).run()


def test_values_that_are_no_numbers(bq):
    """NaN and -inf have no probability, +inf has all, a row of none is its first token's."""
    vocab = 9001
    x, _ = _peaked(10, 9, vocab)
    x[0, ::2] = np.nan
    x[1, 1:] = -INF
    x[2] = -INF
    x[3] = np.nan
    x[4, [5000, 7000]] = INF
    x[5, :] = -INF
    x[5, [8999, 4]] = [1.0, 2.0]
    x[6, 4096:] = -INF
    x[7] = -0.0
    x[7, 1::2] = 0.0
    x[8, :] = np.nan
    x[8, 9000] = -3e38
    for tokens in ([1, 0, 0, 0, 5000, 4, 5000, 8, 9000], [0, 1, 5, 9, 7000, 8999, 0, 9000, 0], [-1, vocab, 1 << 30, -(1 << 31), -5, 4, 3, 2, 1]):
        for top in (0, 1, 3, 64):
            Call(bq, x, tokens, None, top).run()
            Call(bq, x, tokens, 0.6, top).run()


def test_nearly_sure_rows(bq):
    """The first token far ahead: its log p and the entropy are tiny, and keep their relative precision."""
    vocab = 20000
    x = np.random.default_rng(11).standard_normal((6, vocab)).astype(np.float32)
    for r, lead in enumerate((12, 20, 30, 45, 60, 90)):
        x[r, 12345] = lead
    got = Call(bq, x, [12345] * 6, None, 2).run()
    assert (got["logprob"] < 0).all() and (got["entropy"] > 0).all()
    # two first tokens
    x[:, 777] = x[:, 12345]
    Call(bq, x, [777, 12345] * 3, None, 2).run()


def test_outputs_on_their_own(bq):
    x, _ = _peaked(12, 3, 5000)
    for want in (("logprob",), ("rank",), ("entropy",), ("top_tokens",), ("top_logprobs",), ("entropy", "top_tokens"), ("logprob", "top_logprobs")):
        Call(bq, x, [7, 8, 9], None, 6 if "top" in want[-1] else 0, want=want).run()


def test_many_rows(bq):
    x, rng = _peaked(13, 300, 1500)
    Call(bq, x, rng.integers(0, 1500, 300), rng.uniform(0.5, 1.5, 300), 3, ld=1501).run()


def test_agrees_with_the_sampler(bq):
    """Greedy draws are the first alternatives, tokens of rank 0."""
    x, _ = _peaked(14, 8, 50000)
    g = torch.from_numpy(x).cuda()
    out, zero = torch.zeros(8, dtype=torch.int32, device="cuda"), torch.zeros(8, device="cuda")
    bq.Sampler(g, out, zero, temperature=zero).run()
    rank, tops = torch.full((8,), -1, dtype=torch.int32, device="cuda"), torch.zeros((8, 4), dtype=torch.int32, device="cuda")
    bq.LogProbs(g, tokens=out, rank=rank, top_tokens=tops).run()
    assert (rank == 0).all() and torch.equal(tops[:, 0], out)


def test_offsets_past_32_bits(bq):
    """Rows more than 2^32 bytes, and more than 2^31 logits, into the buffer."""
    rows, vocab, ld = 2100, 8, 1 << 20
    buf = torch.empty((rows, ld), device="cuda")
    buf[:, :vocab] = 0
    buf[-1, 5] = 3.0
    lp, tops = torch.zeros(rows, device="cuda"), torch.zeros((rows, 2), dtype=torch.int32, device="cuda")
    bq.LogProbs(buf[:, :vocab], tokens=torch.full((rows,), 5, dtype=torch.int32, device="cuda"), logprob=lp, top_tokens=tops).run()
    assert abs(lp[0].item() + np.log(8)) <= 1e-6 and abs(lp[-1].item() + np.log1p(7 * np.exp(-3.0))) <= 1e-6
    assert tops[0].tolist() == [0, 1] and tops[-1].tolist() == [5, 0]


def test_captured_and_replayed(bq):
    x, _ = _peaked(15, 6, 20000)
    c = Call(bq, x, [1, 2, 3, 4, 5, 6], 0.8, 20)
    c.run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.op.run()
    for step in range(4):
        c.host, rng = _peaked(16 + step, 6, 20000)
        c.tokens = rng.integers(0, 20000, 6).astype(np.int32)
        c.dev.copy_(torch.from_numpy(c.host))
        c.op._keep[1].copy_(torch.from_numpy(c.tokens))
        c.op.work.fill_(0xFF)
        graph.replay()
        torch.cuda.synchronize()
        c.check()
        first = {k: v.clone() for k, v in c.out.items()}
        c.op.run()
        torch.cuda.synchronize()
        assert all(torch.equal(first[k], v) for k, v in c.out.items())


def test_two_calls_on_two_streams(bq):
    calls = [Call(bq, _peaked(30 + i, 40, 30000)[0], list(range(40)), None, 20) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(3):
        for c, st in zip(calls, streams):
            with torch.cuda.stream(st):
                c.op.run()
    torch.cuda.synchronize()
    for c in calls:
        c.check()


def test_refusals(bq):
    x = torch.zeros((3, 100), device="cuda")
    lp, tops = torch.full((3,), 7.0, device="cuda"), torch.full((3, 2), 7, dtype=torch.int32, device="cuda")
    op = bq.LogProbs(x, tokens=torch.zeros(3, dtype=torch.int32, device="cuda"), logprob=lp, top_tokens=tops)
    L, s = bq.load(), op.struct
    call = lambda: L.bq_logprobs(ctypes.byref(s), None)

    def refused(code, **fields):
        keep = {f: getattr(s, f) for f in fields}
        for f, v in fields.items():
            setattr(s, f, v)
        assert call() == code, (fields, call())
        for f, v in keep.items():
            setattr(s, f, v)
    E, N = bq.BQ_EINVAL, bq.BQ_UNSUPPORTED
    for f in (dict(rows=-1), dict(vocab=0), dict(ld=99), dict(top=-1), dict(tokens=None), dict(logits=None), dict(logits=s.logits + 2), dict(work=None),
              dict(work=s.work + 8), dict(work_bytes=s.work_bytes - 1), dict(logprob=None, top=0), dict(logprob=None, top_tokens=None)):
        refused(E, **f)
    for f in (dict(vocab=(1 << 20) + 1, ld=1 << 21), dict(rows=65536), dict(top=65)):
        refused(N, **f)
    assert L.bq_logprobs(None, None) == E
    s.rows = 0
    assert call() == bq.BQ_OK
    torch.cuda.synchronize()
    assert (lp == 7.0).all() and (tops == 7).all()
    W = L.bq_logprobs_workspace_bytes
    assert W(3, 100, 2) == s.work_bytes and W(0, 100, 2) == W(3, 0, 2) == W(3, 100, 65) == W(3, 100, -1) == W(3, (1 << 20) + 1, 2) == 0

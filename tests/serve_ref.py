"""64-bit references of the serving operators (CPU, torch.float64), and pages
of the paged cache packed from the layout's address formulas (include/bq.h)."""
import numpy as np
import torch

NAN_BF16 = 0x7FC0


def addr_bf16(P, D, t, d, value):
    """Index (in values) of token t, dim d among a head's keys or values."""
    return P * D + (t // 8 * D + d) * 8 + t % 8 if value else (d // 8 * P + t) * 8 + d % 8


def addr_q8(P, D, t, d, value):
    """(index of the code in bytes, index of the scale in bytes) from a head's start."""
    if value:
        code = P * D + ((t // 8 * (D // 32) + d // 32) * 16 + d % 16) * 16 + d // 16 % 2 * 8 + t % 8
    else:
        code = ((d // 64 * 4 + d // 8 % 4) * P + t) * 16 + d // 32 % 2 * 8 + d % 8
    return code, 2 * P * D + 2 * ((D // 32 if value else 0) * P + d // 32 * P + t)


def bf16(x):
    return x.float().to(torch.bfloat16)


def quant(x):
    """codes, scales (bf16) of [..., D] fp32, per 32 values."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    d = bf16(g.abs().amax(-1) / 127)
    inv = torch.where(d > 0, 1 / d.float(), torch.zeros(()))
    return (g * inv[..., None]).round().clamp(-127, 127).to(torch.int8).reshape(x.shape), d


def power(x):
    """2^e of the largest magnitude over the last dimension, in [1, 2) 2^e."""
    m = x.abs().amax(-1, keepdim=True).double()
    return torch.where(m > 0, torch.exp2(torch.floor(torch.log2(m.clamp(min=1e-300)))), torch.ones((), dtype=torch.float64))


def half_keys(codes, scales):
    """q8 keys rounded to fp16 (fp64 out): a token's scales over the power of two of its largest are rounded
    to fp16, and so are their products with the codes."""
    p = power(scales.float())
    s = (scales.double() / p).half().repeat_interleave(32, -1)
    return (codes.double() * s.double()).half().double() * p


def half_rows(q):
    """Query rows [.., D] rounded to fp16 over a power of two of their largest value."""
    p = power(q.float()) / 16
    return (q.double() / p).half().double() * p


class Pages:
    """A cache built on the CPU: every byte that holds no token of a sequence is NaN (bf16 pages and q8
    scales) or an extreme code, so a kernel that lets one count gives NaN."""

    def __init__(self, kv_type, heads, D, P, n_seq, max_pages, seed, spare=2):
        self.kv, self.H, self.D, self.P = kv_type, heads, D, P
        self.rng = np.random.default_rng(seed)
        self.n_pages = n_seq * max_pages + spare
        self.head_bytes = 4 * P * D if kv_type == "bf16" else 2 * P * D + P * D // 8
        raw = np.empty((self.n_pages, heads, self.head_bytes // 2), np.uint16)
        raw[:] = NAN_BF16
        self.raw = torch.from_numpy(raw.view(np.uint8).copy())
        if kv_type == "q8":
            self.raw[:, :, : 2 * P * D] = 0x81
        self.table = torch.from_numpy(self.rng.permutation(self.n_pages)[: n_seq * max_pages].reshape(n_seq, max_pages)
                                      .astype(np.int32))
        self.k, self.v = {}, {}
        self.kh = {}  # keys as the prefill attention's products take them

    def put(self, seq, k, v):
        """Tokens 0..n-1 of sequence seq: k and v fp32 [n, H, D]; what the cache then stands for is kept (fp64)."""
        n, P, D = k.shape[0], self.P, self.D
        t = torch.arange(n)[:, None, None]
        h = torch.arange(self.H)[None, :, None]
        d = torch.arange(D)[None, None, :]
        page = self.table[seq][(torch.arange(n) // P)].long()[:, None, None]
        for value, x, keep in ((0, k, self.k), (1, v, self.v)):
            if self.kv == "bf16":
                x = bf16(x)
                if not value:
                    self.kh[seq] = x.double()
                self.raw.view(torch.bfloat16)[page, h, addr_bf16(P, D, t % P, d, value)] = x
                keep[seq] = x.double()
            else:
                c, s = quant(x)
                if not value:
                    self.kh[seq] = half_keys(c, s)
                code, scale = addr_q8(P, D, t % P, d, value)
                self.raw.view(torch.int8)[page, h, code] = c
                sd = s.repeat_interleave(32, -1)
                self.raw.view(torch.bfloat16)[page, h, scale // 2] = sd
                keep[seq] = c.double() * sd.double()

    def cache(self, bq):
        return bq.KvCache(self.raw.reshape(self.n_pages, -1).cuda(), self.table.cuda(),
                          self.kv, self.H, self.D, self.P)


def attention(q, k, v, pos, scale, window=0, sinks=0, hidden=None):
    """q fp64 [R, Hq, D] at positions pos [R]; k, v fp64 [T, H, D].  Returns (out, bound): bound[R, Hq, D] is
    sum_j p_j |v_j|, and A[R, Hq] the largest scale * sum |q_i k_ij| of a visible token, which errors scale with."""
    R, Hq, D = q.shape
    T, H, _ = k.shape
    out = torch.zeros((R, Hq, D), dtype=torch.float64)
    bound, A = out.clone(), torch.zeros((R, Hq), dtype=torch.float64)
    tok = torch.arange(T)
    for r in range(R):
        see = tok <= pos[r]
        if window:
            see &= (tok > pos[r] - window) | (tok < sinks)
        if hidden is not None:
            see &= ~hidden
        if not see.any():
            continue
        for h in range(H):
            ks, vs = k[see, h], v[see, h]
            qs = q[r, h * (Hq // H):(h + 1) * (Hq // H)]
            w = torch.softmax(scale * (qs @ ks.T), 1)
            sl = slice(h * (Hq // H), (h + 1) * (Hq // H))
            out[r, sl] = w @ vs
            bound[r, sl] = w @ vs.abs()
            A[r, sl] = scale * (qs.abs() @ ks.abs().T).amax(1)
    return out, bound, A


def append(q, k, v, pos, cs, rot, qw, kw, eps, interleaved):
    """q [R, Hq, D], k, v [R, H, D] fp64 -> rotated q, k and v; cs fp64 [n_pos, rot]."""
    def head(x, w):
        x = x.clone()
        if w is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
        for i in range(rot // 2):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
            c, s = cs[pos, i][:, None], cs[pos, rot // 2 + i][:, None]
            x[..., a], x[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        return x
    return head(q, qw), head(k, kw), v


def sample_ok(logits, u, temp, k, p, min_p, token, eps=2e-6):
    """Whether `token` is the draw, up to a relative error eps of the running masses and of the cuts."""
    x = logits.astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.lexsort((np.arange(len(x)), -x))
    if not np.isfinite(x[order[0]]) or not temp > 0:
        return token == order[0]
    e = np.exp((x[order] - x[order[0]]) / temp)
    n_k = k if 0 < k < len(x) else len(x)
    cum = np.cumsum(e)
    z = cum[n_k - 1]
    rank = int(np.nonzero(order == token)[0][0])

    def kept(sign):  # kept tokens with the cuts moved by eps
        ex = cum - e
        ok = (np.arange(len(x)) < n_k) & (e >= min_p * (1 + sign * eps))
        if p < 1:
            ok &= ex < p * z - sign * eps * z
        ok[0] = True
        return len(ok) if ok.all() else int(np.argmin(ok))
    for n in range(kept(1), kept(-1) + 1):
        m = cum[n - 1]
        if rank < n and cum[rank] >= u * m - eps * m and cum[rank] - e[rank] <= u * m + eps * m and e[rank] > 0:
            return True
    return False

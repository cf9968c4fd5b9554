"""The serving operators around the quantized matmuls, as cases that can be timed and checked.

Four operators of libbq, called as a decode or prompt step calls them:

  append   per-head norm and rotation of a step's queries and keys, and the step's K and V
           into the pages of a key-value cache (bf16, or q8: int8 codes with one bf16 scale
           per 32 values)
  decode   attention of 1..8 new tokens per sequence over that cache
  prefill  attention of a prompt chunk (a ragged batch of them) over that cache
  sample   a token per row of logits: temperature, top-k, top-p, min-p, from a given uniform number

Sizes: attention width 4096 = 32 heads of 128 over 4 key-value heads (the QKV projection's 5120
outputs), vocabulary 131072, prompt chunks of 512 to 8192 rows, as in the benchmark and the tests;
the others are generic.

Cache pages.  One page holds `P` tokens of every key-value head; per head its keys, then its values:
  bf16  K [D/8][P][8]                      V [P/8][D][8]
  q8    K codes [D/64][4][P][2][8]         (dim 64 c + 32 u + 8 g + i at [c][g][token][u][i])
        V codes [P/8][D/32][16][2][8]      (token 8 t + i, dim 32 c + 16 u + m at [t][c][m][u][i])
        K scales bf16 [D/32][P], V scales bf16 [D/32][P]
"""
import importlib
import math
import random

import torch

own = False

BF16, F32 = torch.bfloat16, torch.float32


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _append(rows, n_seq, ctx, q_heads=32, kv_heads=4, D=128, P=64, kv="bf16", q="f32", norm=True, rot=None,
            inter=False):
    return {"op": "append", "rows": rows, "n_seq": n_seq, "ctx": ctx, "q_heads": q_heads, "kv_heads": kv_heads, "D": D,
            "P": P, "kv": kv, "q": q, "norm": norm, "rot": D if rot is None else rot, "inter": inter}


def _attn(op, n_seq, rows, length, q_heads=32, kv_heads=4, D=128, P=64, kv="bf16", q="f32", out="f32", window=0,
          sinks=0, ragged=False):
    # length: decode: tokens in the cache; prefill: tokens before the chunk
    return {"op": op, "n_seq": n_seq, "rows": rows, "len": length, "q_heads": q_heads, "kv_heads": kv_heads, "D": D,
            "P": P, "kv": kv, "q": q, "out": out, "window": window, "sinks": sinks, "ragged": ragged}


def _sample(rows, vocab, temp, k, p, minp):
    return {"op": "sample", "rows": rows, "vocab": vocab, "temp": temp, "k": k, "p": p, "minp": minp}


def listed():
    return [
        # one decoded token's q, k, v: launch latency
        dict(_append(1, 1, 4096), name="append_token"),
        # a batch of 47 sequences, one token each, into a q8 cache, rotation over half of each head
        dict(_append(47, 47, 8192, P=16, kv="q8", rot=64), name="append_batch47_q8"),
        # a long prompt's rows, queries in bf16 for the prefill attention
        dict(_append(8192, 1, 0, q="bf16"), name="append_prompt8192"),
        # one token of a short chat: latency
        dict(_attn("decode", 1, 1, 777), name="decode_1x777"),
        # a serving batch of 32 sequences of up to 16384 tokens
        dict(_attn("decode", 32, 1, 16384, ragged=True), name="decode_32x16384"),
        # one long document in a q8 cache: the split over the length
        dict(_attn("decode", 1, 1, 131072, kv="q8"), name="decode_1x131072_q8"),
        # speculative verify: five draft tokens of eight sequences, window with sinks, 64-wide heads
        dict(_attn("decode", 8, 5, 9001, D=64, q_heads=32, kv_heads=8, P=16, q="bf16", out="bf16", window=4096,
                   sinks=4), name="verify5_8x9001_window"),
        # a 512-row prompt chunk
        dict(_attn("prefill", 1, 512, 0, q="bf16", out="bf16"), name="prefill_512"),
        # a whole 8192-row prompt
        dict(_attn("prefill", 1, 8192, 0, q="bf16", out="bf16"), name="prefill_8192"),
        # five ragged chunks over earlier tokens, q8 cache, window with sinks
        dict(_attn("prefill", 5, 700, 6000, P=32, kv="q8", q="f32", out="bf16", window=2048, sinks=16, ragged=True),
             name="prefill_ragged5_q8_window"),
        # the next token of one sequence
        dict(_sample(1, 131072, 0.8, 40, 0.95, 0.05), name="sample_1"),
        # a batch's next tokens, nucleus only
        dict(_sample(64, 131072, 0.7, 0, 0.9, 0.0), name="sample_64_top_p"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    kv_heads = rng.choice([1, 2, 4, 8])
    return kv_heads * rng.choice([1, 3, 4, 5, 7, 8]), kv_heads


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "prefill", "prefill", "sample"])
    if op == "sample":
        k = rng.choice([0, 1, 20, 50, 64])
        vocab = _log_int(rng, 8000, 160000)
        return _sample(_log_int(rng, 1, min(96, (1 << 23) // vocab)), vocab, round(rng.uniform(0.5, 1.0), 3), k,
                       round(rng.uniform(0.5, 0.95), 3) if k == 0 or rng.random() < 0.5 else 1.0,
                       rng.choice([0.0, 0.0, 0.02, 0.1]))
    D = rng.choice([64, 128, 128, 256])
    q_heads, kv_heads = _heads(rng)
    P, kv = rng.choice([16, 32, 64, 128]), rng.choice(["bf16", "q8"])
    if op == "append":
        rows = _log_int(rng, 1, min(4096, (1 << 25) // ((q_heads + 2 * kv_heads) * D)))
        return _append(rows, rows if rows <= 64 and rng.random() < 0.7 else rng.randint(1, min(rows, 4)),
                       _log_int(rng, 64, 16384), q_heads, kv_heads, D, P, kv, rng.choice(["f32", "bf16"]),
                       rng.random() < 0.7, rng.choice([D, D // 2]), rng.random() < 0.4)
    window = rng.choice([0, 0, _log_int(rng, 32, 4096)])
    sinks = 0 if window == 0 else rng.choice([0, 4, rng.randint(1, 64)])
    if op == "decode":
        n_seq = _log_int(rng, 1, 64)
        top = min(131072, (1 << 26) // (n_seq * kv_heads * D))
        return _attn(op, n_seq, rng.choice([1, 1, 1, rng.randint(2, 8)]), _log_int(rng, 1, top), q_heads, kv_heads, D, P,
                     kv, rng.choice(["f32", "bf16"]), rng.choice(["f32", "bf16"]), window, sinks, rng.random() < 0.5)
    n_seq = rng.randint(1, 6)
    rows = _log_int(rng, 9, (1 << 18) // (n_seq * D))
    return _attn(op, n_seq, rows, rng.choice([0, _log_int(rng, 1, 8192 // n_seq)]), min(q_heads, 32), kv_heads, D, P, kv,
                 rng.choice(["f32", "bf16"]), "bf16", window, sinks, rng.random() < 0.5)


def _spread(case, n, top, salt):
    """n lengths of at most `top` for a ragged batch (the first one is `top`), from the case alone."""
    if not case["ragged"]:
        return [top] * n
    rng = random.Random(n * 7919 + top * 31 + salt)
    return [top] + [rng.randint((top + 3) // 4, top) for _ in range(n - 1)]


def _lengths(case):
    """(query rows, tokens in the cache) of each sequence, the new rows among the tokens."""
    n = case["n_seq"]
    if case["op"] == "decode":
        return [case["rows"]] * n, _spread(case, n, case["len"], 1)
    rows, past = _spread(case, n, case["rows"], 2), _spread(case, n, case["len"], 3)
    return rows, [r + p for r, p in zip(rows, past)]


def _pairs(case):
    """Visible (query, token) pairs and tokens that any query sees, over the batch (per head)."""
    w, sinks, pairs, tokens = case["window"], case["sinks"], 0, 0
    for r, n in zip(*_lengths(case)):
        first = max(0, n - r)
        for p in range(first, n):
            lo = max(0, p - w + 1) if w else 0
            pairs += p + 1 - lo + min(sinks, lo)
        lo = max(0, first - w + 1) if w else 0
        tokens += n - lo + min(sinks, lo)
    return pairs, tokens


_WIDTH = {"f32": 4, "bf16": 2}


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + 24 * case["rows"], "flops": 4 * n}
    D, Hq, Hk = case["D"], case["q_heads"], case["kv_heads"]
    cached = 2 * D * Hk * (2 if case["kv"] == "bf16" else 1 + 2 / 32)  # bytes of one token in the cache
    if case["op"] == "append":
        r = case["rows"]
        read_back = cached + 4 * D * Hk if case["kv"] == "q8" else 0
        return {"bytes": r * (4 * D * (Hq + 2 * Hk) + 4 * case["rot"] + _WIDTH[case["q"]] * D * Hq + cached + read_back),
                "flops": 8 * r * D * (Hq + Hk)}
    pairs, tokens = _pairs(case)
    rows = sum(_lengths(case)[0])
    return {"bytes": tokens * cached + rows * Hq * D * (_WIDTH[case["q"]] + _WIDTH[case["out"]]),
            "flops": 4 * D * Hq * pairs}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed(seed * 1009 + salt)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _table(g, n_seq, tokens, P):
    """A block table of pages in random order, and the number of pages."""
    per = (max(tokens) + P - 1) // P
    n = n_seq * per + 3
    return torch.randperm(n, generator=g, device="cuda")[: n_seq * per].reshape(n_seq, per).int(), n


def _page_bytes(case):
    return case["kv_heads"] * case["P"] * case["D"] * 4 if case["kv"] == "bf16" else \
        case["kv_heads"] * (2 * case["P"] * case["D"] + case["P"] * case["D"] // 8)


def _random_pages(case, n, g):
    """Pages whose tokens have Gaussian(0, 1) keys and values."""
    H, P, D = case["kv_heads"], case["P"], case["D"]
    if case["kv"] == "bf16":
        return torch.randn((n, H * 2 * P * D), generator=g, device="cuda", dtype=BF16).view(torch.uint8)
    # Gaussian codes on scales as 32 Gaussian values have them
    codes = torch.randn((n, H, 2 * P * D), generator=g, device="cuda", dtype=BF16).mul_(50).round_().clamp_(-127, 127)
    scale = torch.rand((n, H, P * D // 16), generator=g, device="cuda").mul_(0.01).add_(0.015).to(BF16)
    return torch.cat([codes.to(torch.int8).view(torch.uint8), scale.view(torch.uint8)], 2).reshape(n, -1)


def prepare(case, seed):
    g = _gen(seed, 1)
    s = {"case": case}
    if case["op"] == "sample":
        R, V = case["rows"], case["vocab"]
        logits = torch.randn((R, V), generator=g, device="cuda") * 1.5
        few = torch.randint(0, V, (R, 40), generator=g, device="cuda")  # the tokens that the context calls for
        logits.scatter_add_(1, few, torch.rand((R, 40), generator=g, device="cuda") * 9 + 9)
        s.update(logits=logits, u=torch.rand(R, generator=g, device="cuda"),
                 temp=case["temp"] + 0.2 * torch.rand(R, generator=g, device="cuda"),
                 top_k=torch.full((R,), case["k"], dtype=torch.int32, device="cuda"),
                 top_p=torch.full((R,), case["p"], device="cuda"), min_p=torch.full((R,), case["minp"], device="cuda"),
                 out=torch.zeros(R, dtype=torch.int32, device="cuda"))
        return s
    Hq, Hk, D, P = case["q_heads"], case["kv_heads"], case["D"], case["P"]
    if case["op"] == "append":
        R, n = case["rows"], case["n_seq"]
        rng = random.Random(seed * 31 + 7)
        per = [R // n + (i < R % n) for i in range(n)]
        start = [rng.randint(0, case["ctx"]) for _ in range(n)]
        table, pages = _table(g, n, [case["ctx"] + b for b in per], P)
        qkv = torch.randn((R, (Hq + 2 * Hk) * D), generator=g, device="cuda") * 3  # the projections' rows, side by side
        q, k, v = qkv[:, : Hq * D], qkv[:, Hq * D : (Hq + Hk) * D], qkv[:, (Hq + Hk) * D :]
        n_pos = case["ctx"] + max(per)
        half = case["rot"] // 2
        ang = torch.arange(n_pos, device="cuda", dtype=torch.float64)[:, None] * \
            (10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half))
        s.update(q=q, k=k, v=v, table=table, pages=torch.zeros((pages, _page_bytes(case)), dtype=torch.uint8, device="cuda"),
                 rope=torch.cat([ang.cos(), ang.sin()], 1).float(),
                 seq=_ints([i for i in range(n) for _ in range(per[i])]),
                 pos=_ints([start[i] + j for i in range(n) for j in range(per[i])]),
                 qw=1 + 0.2 * torch.randn(D, generator=g, device="cuda") if case["norm"] else None,
                 kw=1 + 0.2 * torch.randn(D, generator=g, device="cuda") if case["norm"] else None,
                 q_out=torch.zeros((R, Hq * D), dtype=BF16 if case["q"] == "bf16" else F32, device="cuda"),
                 k_out=torch.zeros((R, Hk * D), dtype=BF16, device="cuda"),
                 v_out=torch.zeros((R, Hk * D), dtype=BF16, device="cuda"))
        return s
    rows, tokens = _lengths(case)
    table, pages = _table(g, case["n_seq"], tokens, P)
    total = sum(rows)
    q = torch.randn((total, Hq * D), generator=g, device="cuda") * 2
    s.update(q=q.to(BF16) if case["q"] == "bf16" else q, table=table, pages=_random_pages(case, pages, g),
             kv_len=_ints(tokens), row0=_ints([sum(rows[:i]) for i in range(len(rows) + 1)]), max_rows=max(rows),
             max_len=max(tokens), scale=1 / math.sqrt(D),
             out=torch.zeros((total, Hq * D), dtype=BF16 if case["out"] == "bf16" else F32, device="cuda"))
    return s


# ---------------------------------------------------------------------------
# the plain forms (32 bits)
# ---------------------------------------------------------------------------
def _unpack(case, pages):
    """The values that pages [..., page bytes] hold: K and V, fp32 [..., heads, P, D]."""
    H, P, D = case["kv_heads"], case["P"], case["D"]
    lead = pages.shape[:-1]
    if case["kv"] == "bf16":
        kv = pages.view(BF16).reshape(-1, H, 2, P * D)
        k = kv[:, :, 0].reshape(-1, H, D // 8, P, 8).permute(0, 1, 3, 2, 4)
        v = kv[:, :, 1].reshape(-1, H, P // 8, D, 8).permute(0, 1, 2, 4, 3)
        return k.reshape(*lead, H, P, D).float(), v.reshape(*lead, H, P, D).float()
    b = pages.reshape(-1, H, pages.shape[-1] // H)
    codes, scale = b[..., : 2 * P * D].contiguous().view(torch.int8), b[..., 2 * P * D :].contiguous().view(BF16).float()
    k = codes[..., : P * D].reshape(-1, H, D // 64, 4, P, 2, 8).permute(0, 1, 4, 2, 5, 3, 6).reshape(-1, H, P, D // 32, 32)
    v = codes[..., P * D :].reshape(-1, H, P // 8, D // 32, 16, 2, 8).permute(0, 1, 2, 6, 3, 5, 4).reshape(-1, H, P, D // 32, 32)
    ks, vs = scale.reshape(-1, H, 2, D // 32, P).transpose(-1, -2).unbind(2)
    return (k * ks[..., None]).reshape(*lead, H, P, D), (v * vs[..., None]).reshape(*lead, H, P, D)


def _q8(x):
    """Codes and bf16 scales of rows of 32-value groups."""
    x = x.unflatten(-1, (-1, 32))
    d = (x.abs().amax(-1) / 127).to(BF16)
    inv = torch.where(d > 0, 1 / d.float(), 0)
    return (x * inv[..., None]).round().clamp(-127, 127).to(torch.int8), d


def _plain_append(s):
    case = s["case"]
    H, P, D, rot = case["kv_heads"], case["P"], case["D"], case["rot"]
    cs = s["rope"][s["pos"].long()]
    c, sn = cs[:, None, : rot // 2], cs[:, None, rot // 2 :]

    def head(x, w):
        x = x.unflatten(1, (-1, D))
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
        r = x[..., :rot]
        a, b = (r[..., 0::2], r[..., 1::2]) if case["inter"] else (r[..., : rot // 2], r[..., rot // 2 :])
        y = (a * c - b * sn, b * c + a * sn)
        return torch.cat([torch.stack(y, -1).flatten(-2) if case["inter"] else torch.cat(y, -1), x[..., rot:]], -1)

    q, k, v = head(s["q"], s["qw"]), head(s["k"], s["kw"]), s["v"].unflatten(1, (-1, D))
    s["q_out"].copy_(q.flatten(1))
    page, t = s["table"][s["seq"].long(), (s["pos"] // P).long()].long(), (s["pos"] % P).long()
    if case["kv"] == "bf16":
        pages = s["pages"].view(BF16).view(-1, H, 2, P * D)
        pages[:, :, 0].view(-1, H, D // 8, P, 8)[page, :, :, t] = k.unflatten(-1, (-1, 8)).to(BF16)
        pages[:, :, 1].view(-1, H, P // 8, D, 8)[page, :, t // 8, :, t % 8] = v.to(BF16)
        return {"q": s["q_out"], "pages": s["pages"].view(BF16)}
    (kc, kd), (vc, vd) = _q8(k), _q8(v)
    b = s["pages"].view(-1, H, s["pages"].shape[1] // H)
    codes, scale = b.view(torch.int8), b.view(BF16)[..., P * D :].unflatten(-1, (2, D // 32, P))
    codes[..., : P * D].unflatten(-1, (D // 64, 4, P, 2, 8))[page, :, :, :, t] = \
        kc.reshape(-1, H, D // 64, 2, 4, 8).transpose(3, 4)
    codes[..., P * D : 2 * P * D].unflatten(-1, (P // 8, D // 32, 16, 2, 8))[page, :, t // 8, :, :, :, t % 8] = \
        vc.reshape(-1, H, D // 32, 2, 16).transpose(3, 4)
    scale[:, :, 0][page, :, :, t] = kd
    scale[:, :, 1][page, :, :, t] = vd
    s["k_out"].copy_((kc * kd.float()[..., None]).flatten(1))
    s["v_out"].copy_((vc * vd.float()[..., None]).flatten(1))
    return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}


def _plain_attention(s):
    case = s["case"]
    Hq, H, D = case["q_heads"], case["kv_heads"], case["D"]
    n, R = case["n_seq"], s["max_rows"]
    rows = s["row0"][1:] - s["row0"][:-1]
    i = torch.arange(R, device="cuda")
    live = i[None] < rows[:, None]                               # [n, R]: a batch of R rows each, some of them padding
    at = torch.where(live, s["row0"][:-1, None] + i, 0).long()
    q = s["q"].float()[at].reshape(n, R, H, Hq // H, D).permute(0, 2, 3, 1, 4).reshape(n, H, -1, D)
    k, v = (x.permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, : s["max_len"]] for x in _unpack(case, s["pages"][s["table"].long()]))
    j = torch.arange(k.shape[2], device="cuda")
    p = (s["kv_len"] - rows)[:, None] + i                        # each row's position
    see = j <= p[..., None]
    if case["window"]:
        see &= (j > p[..., None] - case["window"]) | (j < case["sinks"])
    see = (see & live[..., None])[:, None, None]                 # [n, 1, 1, R, T]
    x = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(s["scale"]).unflatten(2, (Hq // H, R))
    x = x.masked_fill_(~see, -math.inf)
    m = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(m == -math.inf, 0, m)).exp_()
    z = x.sum(-1, keepdim=True)
    o = torch.matmul(x.flatten(2, 3), v).unflatten(2, (Hq // H, R)) / torch.where(z > 0, z, 1)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, R, Hq * D)
    s["out"].copy_(o[live])
    return s["out"]


def _plain_sample(s):
    x, order = torch.sort(s["logits"], dim=1, descending=True, stable=True)
    e = ((x - x[:, :1]) / s["temp"][:, None]).exp()
    rank = torch.arange(x.shape[1], device="cuda")
    k = torch.where(s["top_k"] > 0, s["top_k"], x.shape[1])[:, None]
    e = torch.where(rank < k, e, 0)
    cum = e.cumsum(1)
    keep = (rank < k) & (cum - e < s["top_p"][:, None] * e.sum(1, keepdim=True)) & (e >= s["min_p"][:, None])
    keep[:, 0] = True
    n = keep.sum(1, keepdim=True)
    target = s["u"][:, None] * cum.gather(1, n - 1)
    pick = torch.minimum((cum <= target).sum(1, keepdim=True), n - 1)
    s["out"].copy_(order.gather(1, pick)[:, 0])
    return s["out"]


# ---------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------
def _handle(s):
    """What a user's program keeps over the calls on the same buffers."""
    if "handle" not in s:
        bq, case = importlib.import_module("bruce-engine_amd.bq"), s["case"]
        if case["op"] == "sample":
            s["handle"] = bq.Sampler(s["logits"], s["out"], s["u"], temperature=s["temp"], top_k=s["top_k"],
                                     top_p=s["top_p"], min_p=s["min_p"])
            return s["handle"]
        kv = s["kv"] = bq.KvCache(s["pages"], s["table"], case["kv"], case["kv_heads"], case["D"], case["P"])
        if case["op"] == "append":
            s["handle"] = bq.Append(kv, s["q"], s["k"], s["v"], s["pos"], s["q_out"], seq=s["seq"], q_weight=s["qw"],
                                    k_weight=s["kw"], eps=1e-6, rope=s["rope"], interleaved=case["inter"])
        else:
            s["handle"] = bq.Attention(kv, s["q"], s["out"], s["kv_len"], scale=s["scale"], window=case["window"],
                                       sinks=case["sinks"], max_len=s["max_len"], max_rows=s["max_rows"],
                                       row0=s["row0"] if case["op"] == "prefill" else None)
    return s["handle"]


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"append": _plain_append, "sample": _plain_sample}.get(op, _plain_attention)(state)
    h = _handle(state)
    if op == "append":
        h.run()
        if state["case"]["kv"] == "bf16":
            return {"q": state["q_out"], "pages": state["pages"].view(BF16)}
        state["kv"].read(state["pos"], state["k_out"], state["v_out"], seq=state["seq"])
        return {"q": state["q_out"], "k": state["k_out"], "v": state["v_out"]}
    if op == "decode":
        h.decode()
    elif op == "prefill":
        h.prefill()
    else:
        h.run()
    return state["out"]


# ---------------------------------------------------------------------------
# 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _address(case, token, dim, value):
    """Index of one value among a head's values in a page (bf16), or of its code among the codes (q8)."""
    P, D = case["P"], case["D"]
    if case["kv"] == "bf16":
        return P * D + (token // 8 * D + dim) * 8 + token % 8 if value else (dim // 8 * P + token) * 8 + dim % 8
    if value:
        return P * D + ((token // 8 * (D // 32) + dim // 32) * 16 + dim % 16) * 16 + dim // 16 % 2 * 8 + token % 8
    return ((dim // 64 * 4 + dim // 8 % 4) * P + token) * 16 + dim // 32 % 2 * 8 + dim % 8


def _exact_cached(case, pages, table, head, n):
    """K and V of tokens 0..n-1 of one sequence and head, fp64 [n, D]."""
    H, P, D = case["kv_heads"], case["P"], case["D"]
    size = _page_bytes(case) // H
    tok, dim = torch.arange(n, device="cuda")[:, None], torch.arange(D, device="cuda")[None]
    base = (table[(tok // P).long()].long() * H + head) * size
    got = []
    for value in (0, 1):
        at = _address(case, tok % P, dim, value)
        if case["kv"] == "bf16":
            got.append(pages.view(BF16).reshape(-1)[base // 2 + at].double())
        else:
            codes = pages.view(torch.int8).reshape(-1)[base + at].double()
            scale = P * D + (value * (D // 32) + dim // 32) * P + tok % P  # in bf16 units from the head's first byte
            got.append(codes * pages.view(BF16).reshape(-1)[base // 2 + scale].double())
    return got


def _exact_attention(case, s):
    Hq, H, D = case["q_heads"], case["kv_heads"], case["D"]
    G, q = Hq // H, s["q"].double()
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    first = 0
    for b, (r, n) in enumerate(zip(*_lengths(case))):
        pos = torch.arange(n - r, n, device="cuda")[:, None]
        tok = torch.arange(n, device="cuda")[None]
        hidden = tok > pos
        if case["window"]:
            hidden |= (tok <= pos - case["window"]) & (tok >= case["sinks"])
        for h in range(H):
            k, v = _exact_cached(case, s["pages"], s["table"][b], h, n)
            for x in range(h * G, h * G + G):
                a = q[first : first + r, x * D : x * D + D] @ k.T * s["scale"]
                a[hidden] = -math.inf
                m = a.max(1, keepdim=True).values.clamp(min=-1e300)
                a = torch.exp(a - m)
                z = a.sum(1, keepdim=True)
                out[first : first + r, x * D : x * D + D] = torch.where(z > 0, a @ v / z, 0.0)
        first += r
    return out


def _exact_append(case, s):
    H, P, D, half = case["kv_heads"], case["P"], case["D"], case["rot"] // 2
    cs = s["rope"].double()[s["pos"].long()]
    dim = torch.arange(D, device="cuda")
    live = dim < 2 * half
    i = torch.where(live, dim // 2 if case["inter"] else dim % half, 0)
    second = (dim % 2 == 1) if case["inter"] else dim >= half
    step = 1 if case["inter"] else half
    mate = torch.where(live, torch.where(second, dim - step, dim + step), dim)
    co = torch.where(live, cs[:, i], 1.0)[:, None]
    si = torch.where(live, torch.where(second, cs[:, half + i], -cs[:, half + i]), 0.0)[:, None]

    def head(x, w):
        x = x.double().reshape(x.shape[0], -1, D)
        if w is not None:
            x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / D + 1e-6) * w.double()
        return x * co + x[..., mate] * si

    q, k, v = head(s["q"], s["qw"]), head(s["k"], s["kw"]), s["v"].double().reshape(-1, H, D)
    if case["kv"] == "q8":
        out = {"q": q.flatten(1)}
        for name, x in (("k", k), ("v", v)):
            x = x.reshape(-1, H, D // 32, 32)
            d = (x.abs().max(-1).values / 127).float().to(BF16).double()[..., None]
            out[name] = (torch.where(d > 0, torch.round(x / torch.where(d > 0, d, 1)), 0).clamp(-127, 127) * d).flatten(1)
        return out
    pages = torch.zeros((s["pages"].shape[0], H, 2 * P * D), dtype=torch.float64, device="cuda")
    page, t = s["table"][s["seq"].long(), (s["pos"] // P).long()].long(), (s["pos"] % P).long()
    for h in range(H):
        for value, x in ((0, k), (1, v)):
            pages[page[:, None], h, _address(case, t[:, None], dim[None], value)] = x[:, h]
    return {"q": q.flatten(1), "pages": pages.reshape(s["pages"].shape[0], -1)}


def _exact_sample(s):
    logits, u, temp = (s[k].double().cpu() for k in ("logits", "u", "temp"))
    top_p, min_p, top_k = s["top_p"].double().cpu(), s["min_p"].double().cpu(), s["top_k"].cpu()
    picks = []
    for r in range(logits.shape[0]):
        x, order = torch.sort(logits[r], descending=True, stable=True)
        n = int(top_k[r]) or len(x)
        e = torch.exp((x[:n] - x[0]) / temp[r])
        total, run_, kept = float(e.sum()), 0.0, []
        for w in e.tolist():  # the shortest run of the likeliest tokens that holds top_p, none below min_p of the first
            if kept and (run_ >= top_p[r] * total or w < min_p[r]):
                break
            run_ += w
            kept.append(run_)
        picks.append(int(order[min(sum(c <= float(u[r]) * run_ for c in kept), len(kept) - 1)]))
    return torch.tensor(picks, dtype=torch.int32)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, s)
    if case["op"] == "sample":
        return _exact_sample(s)
    return _exact_attention(case, s)

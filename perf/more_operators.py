"""Operators of a batch of many users' requests, as cases that can be timed and checked.

Three operators of libbq, called as a serving program's step calls them:

  shared    attention of 1..8 new tokens per sequence over the paged key-value cache, for sequences in
            groups that share a long prefix (a system prompt, a document), whose tokens lie in the cache once
  lora      low-rank adapters beside a projection: every row has an adapter of its own,
            y[r] = base[r] + scale B (A x[r]), for up to four matrices that share x
  logprobs  of rows of logits: the log probability and the rank of a given token, the entropy, and the
            likeliest tokens with theirs

Sizes: attention width 4096 = 32 heads of 128 over 4 key-value heads, hidden size 2560 with a feed-forward
width of 7168, vocabulary 131072, prompts of up to 8192 rows; the others are generic.

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
def _shared(n_seq, groups, prefix, tail, rows=1, q_heads=32, kv_heads=4, D=128, P=64, kv="bf16", q="f32", out="f32",
            window=0, sinks=0, ragged=False):
    # prefix: tokens that a group shares; tail: the most tokens of a sequence behind them
    return {"op": "shared", "n_seq": n_seq, "groups": groups, "prefix": prefix, "tail": tail, "rows": rows,
            "q_heads": q_heads, "kv_heads": kv_heads, "D": D, "P": P, "kv": kv, "q": q, "out": out, "window": window,
            "sinks": sinks, "ragged": ragged}


def _lora(rows, K, N, rank, adapters, x="q8", mixed=True):
    # N: the parts' widths joined by "+"; mixed: any row may have any adapter, else runs of rows share one
    return {"op": "lora", "rows": rows, "K": K, "N": N, "rank": rank, "adapters": adapters, "x": x, "mixed": mixed}


def _logprobs(rows, vocab, top, temp=1.0):
    return {"op": "logprobs", "rows": rows, "vocab": vocab, "top": top, "temp": temp}


def listed():
    return [
        # four short chats behind one system prompt: latency
        dict(_shared(4, 1, 600, 90, ragged=True), name="shared_4x600"),
        # a batch of 32 questions about one document
        dict(_shared(32, 1, 16384, 512, ragged=True), name="shared_32x16384"),
        # 64 samples of one prompt that have grown long answers, bf16 in and out
        dict(_shared(64, 1, 8192, 2048, q="bf16", out="bf16", ragged=True), name="shared_64x8192_bf16"),
        # 48 sequences behind three system prompts of their applications, q8 cache
        dict(_shared(48, 3, 6001, 1000, kv_heads=8, P=32, kv="q8", ragged=True), name="shared_48_in_3_q8"),
        # speculative verify: five draft tokens of eight sequences, 64-wide heads, window with sinks
        dict(_shared(8, 1, 3500, 1500, rows=5, kv_heads=8, D=64, P=16, q="bf16", out="bf16", window=4096, sinks=4,
                     ragged=True), name="shared_verify5_window"),
        # one request's output projection: latency
        dict(_lora(1, 4096, "2560", 16, 4), name="lora_1"),
        # 32 requests with 12 adapters between them at the q, k, gate and v projections
        dict(_lora(32, 2560, "4096+512+4096+512", 16, 12), name="lora_32_qkv"),
        # prompts of three users in one batch at the gate and up projections
        dict(_lora(4096, 2560, "7168+7168", 32, 3, mixed=False), name="lora_prompt4096_gate_up"),
        # ragged prompts with wide adapters at the down projection, rows as they left an fp32 kernel
        dict(_lora(777, 7168, "2560", 64, 9, x="f32", mixed=False), name="lora_777_down"),
        # one answer's token with its five alternatives
        dict(_logprobs(1, 131072, 5), name="logprobs_1"),
        # a batch's tokens with twenty alternatives at the sampling temperature
        dict(_logprobs(64, 131072, 20, 0.7), name="logprobs_64_top20"),
        # scoring a prompt chunk: its own tokens' log probabilities, and the likeliest beside each
        dict(_logprobs(512, 131072, 1), name="logprobs_512"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["shared", "shared", "lora", "lora", "logprobs"])
    if op == "logprobs":
        vocab = _log_int(rng, 8000, 160000)
        return _logprobs(_log_int(rng, 1, min(512, (1 << 25) // vocab)), vocab, rng.choice([0, 1, 5, 20, 33, 64]),
                         round(rng.uniform(0.5, 1.5), 3))
    if op == "lora":
        parts = rng.choice([1, 1, 2, 3, 4])
        K, N = 32 * _log_int(rng, 16, 288), [16 * _log_int(rng, 16, 512) for _ in range(parts)]
        rows = _log_int(rng, 1, min(8192, (1 << 25) // (K + sum(N))))
        rank = rng.choice([8, 16, 16, 24, 32, 64, 128])
        top = max(1, (1 << 27) // (rank * (parts * K + sum(N))))
        return _lora(rows, K, "+".join(map(str, N)), rank, min(top, rng.choice([1, 2, 7, 16, 64])),
                     rng.choice(["q8", "f32", "bf16"]), rng.random() < (0.9 if rows <= 64 else 0.2))
    D = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    q_heads = kv_heads * rng.choice([1, 3, 4, 5, 8])
    n_seq = _log_int(rng, 1, 64)
    groups = min(n_seq, rng.choice([1, 1, 1, 2, 5]))
    rows = rng.choice([1, 1, 1, rng.randint(2, 8)])
    tail = _log_int(rng, rows, max(rows, min(4096, (1 << 23) // (n_seq * kv_heads * D))))
    prefix = _log_int(rng, 1, max(1, min(32768, (1 << 31) // (n_seq * rows * q_heads * D) - tail,
                                        (1 << 24) // (groups * kv_heads * D))))
    window = rng.choice([0, 0, 0, _log_int(rng, 32, 8192)])
    return _shared(n_seq, groups, prefix, tail, rows, q_heads, kv_heads, D, rng.choice([16, 32, 64, 128]),
                   rng.choice(["bf16", "q8"]), rng.choice(["f32", "bf16"]), rng.choice(["f32", "bf16"]), window,
                   0 if window == 0 else rng.choice([0, 4, rng.randint(1, 64)]), rng.random() < 0.6)


def _plan(case):
    """Of a shared case: each group's first sequence (and one behind the last), its tokens, and every sequence's
    length, from the case alone.  The first group and the first sequence have the largest."""
    n, G = case["n_seq"], case["groups"]
    first, length, own_ = [n * g // G for g in range(G + 1)], [case["prefix"]] * G, [case["tail"]] * n
    if case["ragged"]:
        rng = random.Random(n * 7919 + case["prefix"] * 31 + case["tail"])
        inner = sorted(rng.sample(range(1, n), G - 1))
        first = [0] + inner + [n]
        length = [case["prefix"]] + [rng.randint((case["prefix"] + 1) // 2, case["prefix"]) for _ in range(G - 1)]
        own_ = [case["tail"]] + [rng.randint(min(case["rows"], case["tail"]), case["tail"]) for _ in range(n - 1)]
    group = [max(g for g in range(G) if first[g] <= s) for s in range(n)]
    return first, length, group, [length[group[s]] + own_[s] for s in range(n)]


def _visible(case):
    """Visible (query, token) pairs, and tokens of the cache that some query sees (each prefix once), per head."""
    first, length, group, total = _plan(case)
    w, sinks, rows = case["window"], case["sinks"], case["rows"]
    pairs, seen, reach = 0, 0, {}
    for s, n in enumerate(total):
        for p in range(n - rows, n):
            lo = max(0, p - w + 1) if w else 0
            pairs += p + 1 - lo + min(sinks, lo)
        lo, c = max(0, n - rows - w + 1) if w else 0, length[group[s]]
        seen += n - max(lo, c) + max(0, min(sinks, lo) - c)
        # of the prefix: the sinks and everything from the lowest window's edge on
        reach[group[s]] = min(reach.get(group[s], c), lo)
    for g, lo in reach.items():
        seen += length[g] - min(lo, length[g]) + min(sinks, lo, length[g])
    return pairs, seen


_WIDTH = {"f32": 4, "bf16": 2, "q8": 1 + 4 / 32}


def _used(case):
    """Adapters of the rows, from the case alone."""
    rng = random.Random(case["rows"] * 131 + case["K"] + case["adapters"])
    n = case["adapters"]
    if case["mixed"]:
        return [rng.randrange(n) for _ in range(case["rows"])]
    cuts = sorted(rng.randint(0, case["rows"]) for _ in range(n - 1))
    order = rng.sample(range(n), n)
    return [order[sum(c <= r for c in cuts)] for r in range(case["rows"])]


def work(case):
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + case["rows"] * (16 + 8 * case["top"]), "flops": 6 * n}
    if case["op"] == "lora":
        N, K, r, rank = [int(n) for n in case["N"].split("+")], case["K"], case["rows"], case["rank"]
        weights = len(set(_used(case))) * rank * 2 * (len(N) * K + sum(N))
        return {"bytes": int(r * K * _WIDTH[case["x"]]) + weights + 8 * r * sum(N) + 4 * r,
                "flops": 2 * r * rank * (len(N) * K + sum(N))}
    D, Hq, Hk = case["D"], case["q_heads"], case["kv_heads"]
    cached = 2 * D * Hk * (2 if case["kv"] == "bf16" else 1 + 2 / 32)  # bytes of one token in the cache
    pairs, tokens = _visible(case)
    rows = case["n_seq"] * case["rows"]
    return {"bytes": int(tokens * cached + rows * Hq * D * (_WIDTH[case["q"]] + _WIDTH[case["out"]])),
            "flops": 4 * D * Hq * pairs}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed(seed * 1009 + salt)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


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


def _prepare_shared(case, seed, s):
    g = _gen(seed, 1)
    first, length, group, total = _plan(case)
    P, n = case["P"], case["n_seq"]
    per = (max(total) + P - 1) // P
    # every sequence has pages of its own but for the whole pages of its group's prefix, in any order in the pool
    ids = torch.arange(n * per).reshape(n, per)
    for q in range(n):
        whole = length[group[q]] // P
        ids[q, :whole] = ids[first[group[q]], :whole]
    used, ids = torch.unique(ids, return_inverse=True)
    pages = len(used) + 3
    table = torch.randperm(pages, generator=g, device="cuda")[ids.cuda()].int()
    rows = n * case["rows"]
    q = torch.randn((rows, case["q_heads"] * case["D"]), generator=g, device="cuda") * 2
    s.update(q=q.to(BF16) if case["q"] == "bf16" else q, table=table, pages=_random_pages(case, pages, g),
             kv_len=_ints(total), group0=_ints(first), prefix_len=_ints(length), group=_ints(group), max_len=max(total),
             max_prefix=max(length), scale=1 / math.sqrt(case["D"]),
             out=torch.zeros(q.shape, dtype=BF16 if case["out"] == "bf16" else F32, device="cuda"))


def _prepare_lora(case, seed, s):
    g = _gen(seed, 2)
    R, K, rank, n = case["rows"], case["K"], case["rank"], case["adapters"]
    x = torch.randn((R, K), generator=g, device="cuda")
    if case["x"] == "q8":  # int8 codes with one fp32 scale per 32 values, as the projection read the row
        t = x.reshape(R, K // 32, 32)
        d = t.abs().amax(-1) / 127
        s["x"] = ((t / d[..., None]).round().clamp(-127, 127).to(torch.int8).reshape(R, K), d.contiguous())
    else:
        s["x"] = x.to(BF16) if case["x"] == "bf16" else x
    s["parts"] = []
    for N in (int(v) for v in case["N"].split("+")):
        a = torch.randn((n, rank, K), generator=g, device="cuda").mul_(K ** -0.5).to(BF16)
        b = torch.randn((n, N, rank), generator=g, device="cuda").mul_(0.3).to(BF16)
        base = torch.randn((R, N), generator=g, device="cuda")
        s["parts"].append((a, b, torch.zeros_like(base), base))
    s.update(adapter=_ints(_used(case)), scale=torch.rand(n, generator=g, device="cuda") + 0.5)


def _prepare_logprobs(case, seed, s):
    g = _gen(seed, 3)
    R, V, top = case["rows"], case["vocab"], case["top"]
    logits = torch.randn((R, V), generator=g, device="cuda") * 1.5
    few = torch.randint(0, V, (R, 40), generator=g, device="cuda")  # the tokens that the context calls for
    logits.scatter_add_(1, few, torch.rand((R, 40), generator=g, device="cuda") * 9 + 9)
    tokens = few[:, 0].clone()
    tokens[::5] = torch.randint(0, V, (tokens[::5].shape[0],), generator=g, device="cuda")  # and some that it does not
    s.update(logits=logits, tokens=tokens.int(),
             temp=case["temp"] + 0.1 * torch.rand(R, generator=g, device="cuda") if case["temp"] != 1.0 else None,
             logprob=torch.zeros(R, device="cuda"), rank=torch.zeros(R, dtype=torch.int32, device="cuda"),
             entropy=torch.zeros(R, device="cuda"),
             top_tokens=torch.zeros((R, top), dtype=torch.int32, device="cuda") if top else None,
             top_logprobs=torch.zeros((R, top), device="cuda") if top else None)


def prepare(case, seed):
    s = {"case": case}
    {"shared": _prepare_shared, "lora": _prepare_lora, "logprobs": _prepare_logprobs}[case["op"]](case, seed, s)
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


def _tokens(case, pages, table):
    """K and V [n, heads, tokens, D] of the pages in table [n, pages]."""
    return [x.permute(0, 2, 1, 3, 4).flatten(2, 3) for x in _unpack(case, pages[table.long()])]


def _plain_shared(s):
    """Scores over the prefix (once for a group's rows together) and over each sequence's own tokens, side by side."""
    case = s["case"]
    Hq, H, D, P, R, n = case["q_heads"], case["kv_heads"], case["D"], case["P"], case["rows"], case["n_seq"]
    G, L = Hq // H, s["max_prefix"]
    q = s["q"].float().reshape(n, R, H, G, D).permute(0, 2, 3, 1, 4).reshape(n, H, G * R, D)
    c = s["prefix_len"].long()[s["group"].long()]                       # [n]: shared tokens
    p = (s["kv_len"] - R)[:, None] + torch.arange(R, device="cuda")     # [n, R]: positions

    def see(tok, ok):                                                   # tok [n, T] -> [n, 1, 1, R, T]
        m = ok[:, None] & (tok[:, None] <= p[..., None])
        if case["window"]:
            m &= (tok[:, None] > p[..., None] - case["window"]) | (tok[:, None] < case["sinks"])
        return m[:, None, None]

    j = torch.arange(L, device="cuda").expand(n, L)
    k0, v0 = (x[:, :, :L] for x in _tokens(case, s["pages"], s["table"][s["group0"][:-1].long(), : (L + P - 1) // P]))
    # rows of a group against its prefix: one product a group
    cuts = _plan(case)[0]
    x0 = torch.empty((n, H, G * R, L), device="cuda")
    for g in range(case["groups"]):
        a, b = cuts[g], cuts[g + 1]
        rows = q[a:b].transpose(0, 1).reshape(H, -1, D)
        x0[a:b] = torch.matmul(rows, k0[g].transpose(1, 2).contiguous()).reshape(H, b - a, G * R, L).transpose(0, 1)
    # own tokens: the pages from the prefix' last on
    T = s["max_len"] - int(min(_plan(case)[1])) + P
    at = (c // P)[:, None] + torch.arange((T + P - 1) // P + 1, device="cuda")
    ids = s["table"].gather(1, at.clamp(max=s["table"].shape[1] - 1))
    k1, v1 = _tokens(case, s["pages"], ids)
    tok = (c // P * P)[:, None] + torch.arange(k1.shape[2], device="cuda")
    x1 = torch.matmul(q, k1.transpose(2, 3).contiguous())
    x0 = x0.mul_(s["scale"]).unflatten(2, (G, R)).masked_fill_(~see(j, j < c[:, None]), -math.inf)
    x1 = x1.mul_(s["scale"]).unflatten(2, (G, R)).masked_fill_(~see(tok, tok >= c[:, None]), -math.inf)
    m = torch.maximum(x0.amax(-1, keepdim=True), x1.amax(-1, keepdim=True))
    m = torch.where(m == -math.inf, 0, m)
    x0, x1 = x0.sub_(m).exp_(), x1.sub_(m).exp_()
    z = x0.sum(-1, keepdim=True) + x1.sum(-1, keepdim=True)
    o = torch.matmul(x1.flatten(2, 3), v1)
    for g in range(case["groups"]):
        a, b = cuts[g], cuts[g + 1]
        w = x0[a:b].flatten(2, 3).transpose(0, 1).reshape(H, -1, L)
        o[a:b] += torch.matmul(w, v0[g]).reshape(H, b - a, G * R, D).transpose(0, 1)
    o = o.unflatten(2, (G, R)) / torch.where(z > 0, z, 1)
    s["out"].copy_(o.permute(0, 3, 1, 2, 4).reshape(n * R, Hq * D))
    return s["out"]


def _plain_lora(s):
    x = s["x"]
    if s["case"]["x"] == "q8":
        x = (x[0].float().unflatten(1, (-1, 32)) * x[1][..., None]).flatten(1)
    x = x.float()
    for a, b, y, base in s["parts"]:
        y.copy_(base)
        for i in range(s["case"]["adapters"]):
            live = s["adapter"] == i
            d = torch.matmul(torch.matmul(x, a[i].float().t().contiguous()), b[i].float().t().contiguous())
            y.add_(torch.where(live[:, None], d * s["scale"][i], 0))
    return [p[2] for p in s["parts"]]


def _plain_logprobs(s):
    case, z, t = s["case"], s["logits"], s["tokens"].long()[:, None]
    m = z.amax(1, keepdim=True)
    x = z - m if s["temp"] is None else (z - m) / s["temp"][:, None]
    e = x.exp()
    total = e.sum(1, keepdim=True)
    log_z = total.log()
    i = torch.arange(z.shape[1], device="cuda")
    zt = z.gather(1, t)
    s["logprob"].copy_((x.gather(1, t) - log_z)[:, 0])
    s["rank"].copy_(((z > zt) | ((z == zt) & (i < t))).sum(1))
    s["entropy"].copy_((log_z - (e * x).sum(1, keepdim=True) / total)[:, 0])
    if case["top"]:
        order = torch.sort(z, dim=1, descending=True, stable=True)[1][:, : case["top"]]
        s["top_tokens"].copy_(order)
        s["top_logprobs"].copy_(x.gather(1, order) - log_z)
    return _logprob_outputs(s)


def _logprob_outputs(s):
    return {k: s[k] for k in ("logprob", "rank", "entropy", "top_tokens", "top_logprobs") if s[k] is not None}


# ---------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------
def _handle(s):
    """What a user's program keeps over the calls on the same buffers."""
    if "handle" not in s:
        bq, case = importlib.import_module("bruce-engine_amd.bq"), s["case"]
        if case["op"] == "shared":
            kv = bq.KvCache(s["pages"], s["table"], case["kv"], case["kv_heads"], case["D"], case["P"])
            s["handle"] = bq.SharedAttention(kv, s["q"], s["out"], s["kv_len"], s["group0"], s["prefix_len"],
                                             scale=s["scale"], window=case["window"], sinks=case["sinks"],
                                             max_len=s["max_len"], max_prefix=s["max_prefix"])
        elif case["op"] == "lora":
            s["handle"] = bq.Lora(s["x"], s["adapter"], s["parts"], scale=s["scale"])
        else:
            s["handle"] = bq.LogProbs(s["logits"], tokens=s["tokens"], logprob=s["logprob"], rank=s["rank"],
                                      entropy=s["entropy"], top_tokens=s["top_tokens"], top_logprobs=s["top_logprobs"],
                                      temperature=s["temp"])
    return s["handle"]


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"shared": _plain_shared, "lora": _plain_lora, "logprobs": _plain_logprobs}[op](state)
    _handle(state).run()
    if op == "shared":
        return state["out"]
    return [p[2] for p in state["parts"]] if op == "lora" else _logprob_outputs(state)


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


def _exact_cached(case, pages, page, tok, head):
    """K and V of one head's tokens tok [n] in pages page [n], fp64 [n, D]."""
    H, P, D = case["kv_heads"], case["P"], case["D"]
    size = _page_bytes(case) // H
    tok, dim = tok[:, None] % P, torch.arange(D, device="cuda")[None]
    base = (page.long()[:, None] * H + head) * size
    got = []
    for value in (0, 1):
        at = _address(case, tok, dim, value)
        if case["kv"] == "bf16":
            got.append(pages.view(BF16).reshape(-1)[base // 2 + at].double())
        else:
            codes = pages.view(torch.int8).reshape(-1)[base + at].double()
            scale = P * D + (value * (D // 32) + dim // 32) * P + tok  # in bf16 units from the head's first byte
            got.append(codes * pages.view(BF16).reshape(-1)[base // 2 + scale].double())
    return got


def _exact_shared(case, s):
    Hq, H, D, R = case["q_heads"], case["kv_heads"], case["D"], case["rows"]
    G, q = Hq // H, s["q"].double()
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    first, length, group, total = _plan(case)
    for b, n in enumerate(total):
        tok = torch.arange(n, device="cuda")
        shared = tok < length[group[b]]
        page = torch.where(shared, s["table"][first[group[b]]][tok // case["P"]], s["table"][b][tok // case["P"]])
        pos = torch.arange(n - R, n, device="cuda")[:, None]
        hidden = tok[None] > pos
        if case["window"]:
            hidden |= (tok[None] <= pos - case["window"]) & (tok[None] >= case["sinks"])
        for h in range(H):
            k, v = _exact_cached(case, s["pages"], page, tok, h)
            for x in range(h * G, h * G + G):
                a = q[b * R : b * R + R, x * D : x * D + D] @ k.T * s["scale"]
                a[hidden] = -math.inf
                m = a.max(1, keepdim=True).values.clamp(min=-1e300)
                a = torch.exp(a - m)
                z = a.sum(1, keepdim=True)
                out[b * R : b * R + R, x * D : x * D + D] = torch.where(z > 0, a @ v / z, 0.0)
    return out


def _exact_lora(case, s):
    if case["x"] == "q8":
        codes, d = s["x"]
        x = codes.double() * d.double().repeat_interleave(32, 1)
    else:
        x = s["x"].double()
    outs = []
    for a, b, _, base in s["parts"]:
        y = base.double()
        for i in range(case["adapters"]):
            at = torch.nonzero(s["adapter"] == i)[:, 0]
            y[at] += s["scale"][i].double() * (x[at] @ a[i].double().T @ b[i].double().T)
        outs.append(y)
    return outs


def _exact_logprobs(case, s):
    z = s["logits"].double()
    t = torch.ones(z.shape[0], dtype=torch.float64, device="cuda") if s["temp"] is None else s["temp"].double()
    p = z / t[:, None]
    lp = p - torch.logsumexp(p, 1, keepdim=True)
    tok = s["tokens"].long()
    rows = torch.arange(z.shape[0], device="cuda")
    zt = z[rows, tok][:, None]
    before = (z > zt).sum(1) + ((z == zt) & (torch.arange(z.shape[1], device="cuda")[None] < tok[:, None])).sum(1)
    out = {"logprob": lp[rows, tok], "rank": before.int(), "entropy": -(lp.exp() * lp).sum(1)}
    if case["top"]:
        top = torch.argsort(-z, dim=1, stable=True)[:, : case["top"]]
        out.update(top_tokens=top.int(), top_logprobs=lp.gather(1, top))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"shared": _exact_shared, "lora": _exact_lora, "logprobs": _exact_logprobs}[case["op"]](case, s)

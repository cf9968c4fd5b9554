"""Token generation through libbq: prompt chunks, then decoded tokens, with the
library's own attention and sampling around its matmuls.

    python bruce-engine_amd/generate.py [--kv q8] [--tokens 32] [--batch 4] ...

Random weights of a small architecture (or larger, by the options), random
prompts.  What it shows is the wiring a serving program needs:

* one KvCache per attention block, sharing a block table;
* a bq_decode_step whose attention is the library's hook: AttentionPlan holds an
  Append and an Attention per attention block;
* prompts in chunks (BQ rows of one sequence, prefill attention), then all
  sequences together, one token each, as one captured graph replayed per token
  (positions and lengths are device memory, so one graph serves them all);
* Sampler on the logits; its tokens feed the next step without leaving the GPU.
"""
import argparse
import ctypes
import os
import sys

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
if HERE not in sys.path:
    sys.path.insert(0, HERE)

import bq  # noqa: E402
import synth  # noqa: E402


class Config:
    def __init__(self, n_embd=1024, q_heads=8, kv_heads=2, head_dim=128, n_ff=2048, layers=2, vocab=4096,
                 kv_type="bf16", page_tokens=64, window=0, sinks=0):
        self.n_embd, self.q_heads, self.kv_heads, self.head_dim = n_embd, q_heads, kv_heads, head_dim
        self.n_ff, self.layers, self.vocab = n_ff, layers, vocab
        self.kv_type, self.page_tokens, self.window, self.sinks = kv_type, page_tokens, window, sinks
        self.n_attn, self.n_kv = q_heads * head_dim, kv_heads * head_dim


class Model:
    """Random weights: per layer q, k, gate and v (Q5_K, with the W144 repack the prefill GEMMs use), o, gate, up
    (Q5_K), down (Q6_K, W160), the norm weights of q and k, and a Q8_0 head."""

    def __init__(self, c, seed=0):
        import torch
        self.c = c
        g = torch.Generator().manual_seed(seed)
        self.rng = np.random.default_rng(seed)
        vec = lambda n, mean=1.0, std=0.2: (mean + std * torch.randn(n, generator=g)).cuda()
        self.layers = []
        for _ in range(c.layers):
            self.layers.append({
                "qkv": [self._q5(c.n_embd, n) for n in (c.n_attn, c.n_kv, c.n_attn, c.n_kv)],
                "o": self._q5(c.n_attn, c.n_embd), "gate": self._q5(c.n_embd, c.n_ff), "up": self._q5(c.n_embd, c.n_ff),
                "down": self._q6(c.n_ff, c.n_embd), "sgate": vec(c.n_attn), "s_gate": vec(c.n_ff), "s_up": vec(c.n_ff),
                "alpha_a": vec(c.n_embd, 0.5), "alpha_f": vec(c.n_embd, 0.5),
                "q_weight": vec(c.head_dim), "k_weight": vec(c.head_dim),
            })
        self.embed = torch.randn((c.vocab, c.n_embd), generator=g).cuda()
        self.head = bq.quantize_q8s((torch.randn((c.vocab, c.n_embd), generator=g) * 0.3).bfloat16().view(torch.int16).cuda(),
                                    c.n_embd, c.vocab)
        self.scale = vec(c.vocab, 8.0, 0.5)

    def _raw(self, quantize, K, N):
        import torch
        return torch.from_numpy(quantize(self.rng.standard_normal((N, K)).astype(np.float32) * 0.02)).cuda()

    def _q5(self, K, N):
        raw = self._raw(synth.quantize_q5k, K, N)
        rep, rep_min = bq.repack_q5k(raw, K, N)
        return bq.make_weight(raw, bq.TYPE_Q5_K, K, N, rep=rep, rep_min=rep_min)

    def _q6(self, K, N):
        raw = self._raw(synth.quantize_q6k, K, N)
        return bq.make_weight(raw, bq.TYPE_Q6_K, K, N, rep=bq.repack_q6k(raw, K, N))


class Step:
    """A decode step over `rows` rows of the model: buffers, the attention plan over `caches`, and run().  decode:
    row r is the next token of sequence r; otherwise the rows are a chunk of the only sequence of the caches.
    max_len: the most tokens a sequence has in any run (it sizes the attention's workspace and its pieces)."""

    def __init__(self, model, caches, rope, rows, pos, kv_len, max_len, decode):
        import torch
        c, self.model, self.rows = model.c, model, rows
        f32 = lambda *s: torch.zeros(s, device="cuda")
        wide = max(c.n_embd, c.n_attn, c.n_ff)
        self.x, self.proj = f32(rows, c.n_embd), f32(rows, c.n_embd)
        self.q8 = (torch.zeros(rows * wide, dtype=torch.int8, device="cuda"), f32(rows * wide // 32),
                   torch.zeros(rows * wide // 32, dtype=torch.int32, device="cuda"))
        self.logits = f32(rows if rows <= 8 else 1, c.vocab)
        self.qkv = [f32(rows, n) for n in (c.n_attn, c.n_kv, c.n_attn, c.n_kv)]   # q, k, gate, v: one layer's at a time
        self.attn_out = f32(rows, c.n_attn)
        # fp32 queries for the decode attention, bf16 for the prefill attention's products
        self.q = torch.zeros((rows, c.n_attn), dtype=torch.float32 if decode else torch.bfloat16, device="cuda")
        self.pos, self.kv_len = pos, kv_len
        seq = torch.arange(rows, dtype=torch.int32, device="cuda") if decode else None
        ffn = [f32(rows, c.n_ff) for _ in range(2)]
        xdh = torch.zeros((rows, wide // 32), dtype=torch.int16, device="cuda")
        work = torch.empty(8 << 20, dtype=torch.float32, device="cuda")
        P, ptr = ctypes.pointer, lambda t: t.data_ptr()
        blocks, plan, keep = [], [], []
        attn_work = "auto"  # the layers run one after another: the first one's serves all
        for cache, L in zip(caches, model.layers):
            qkv = (bq.Weight * 4)(*L["qkv"])
            outs = (ctypes.c_void_p * 4)(*[ptr(t) for t in self.qkv])
            keep += [qkv, outs]
            b = bq.DecodeBlock()
            b.kind, b.alpha, b.qkv, b.n_qkv, b.qkv_out = bq.BLOCK_ATTN, ptr(L["alpha_a"]), qkv, 4, outs
            b.attn_out, b.attn_gate, b.sgate, b.n_attn, b.o = ptr(self.attn_out), ptr(self.qkv[2]), ptr(L["sgate"]), c.n_attn, P(L["o"])
            blocks.append(b)
            append = bq.Append(cache, self.qkv[0], self.qkv[1], self.qkv[3], pos, self.q, seq=seq, q_weight=L["q_weight"],
                               k_weight=L["k_weight"], rope=rope)
            attention = bq.Attention(cache, self.q, self.attn_out, kv_len, window=c.window, sinks=c.sinks, max_len=max_len,
                                     work=attn_work)
            attn_work = attention.work
            plan.append((append, attention))
            b = bq.DecodeBlock()
            b.kind, b.alpha, b.gate, b.up, b.down = bq.BLOCK_FFN, ptr(L["alpha_f"]), P(L["gate"]), P(L["up"]), P(L["down"])
            b.s_gate, b.s_up, b.n_ff = ptr(L["s_gate"]), ptr(L["s_up"]), c.n_ff
            blocks.append(b)
            plan.append(None)
        blocks[-1].norm_after = 1
        self.blocks = (bq.DecodeBlock * len(blocks))(*blocks)
        st = self.struct = bq.DecodeStep()
        st.n_blocks, st.blocks, st.n_embd, st.rows = len(blocks), self.blocks, c.n_embd, rows
        st.x, st.proj, st.ffn_g, st.ffn_u = ptr(self.x), ptr(self.proj), ptr(ffn[0]), ptr(ffn[1])
        st.xq, st.xd, st.xsum = (ptr(t) for t in self.q8)
        st.head_q8s, st.head_rs, st.vocab, st.logits = ptr(model.head), ptr(model.scale), c.vocab, ptr(self.logits)
        st.xdh, st.work, st.work_bytes = ptr(xdh), ptr(work), work.numel() * 4
        self.plan = bq.AttentionPlan(plan, prefill=not decode)
        self.plan.install(st)
        self._keep = (blocks, keep, ffn, xdh, work, caches, rope, seq)
        self.graph = None

    def capture(self):
        self.graph = bq.DecodeGraph(self.struct)
        self.plan.check()

    def run(self, tokens):
        """Embeds tokens [rows] (device) and runs the step; the logits are in self.logits."""
        import torch
        torch.index_select(self.model.embed, 0, tokens, out=self.x)
        n = self.model.c.n_embd
        bq.norm_q8("norm", self.rows, n, out=self.x, a=self.x, q8=self.q8)
        if self.graph is not None:
            self.graph.launch()
        else:
            bq.decode_enqueue(self.struct)
            self.plan.check()
        return self.logits


class Generator:
    """Sequences over one paged cache per layer: prefill(s, tokens), then decode() rounds over all of them."""

    def __init__(self, model, n_seq, max_len, seed=1):
        import torch
        c, self.model, self.n_seq, self.max_len = model.c, model, n_seq, max_len
        per = (max_len + c.page_tokens - 1) // c.page_tokens
        ids = torch.randperm(n_seq * per, generator=torch.Generator().manual_seed(seed))
        self.table = ids.reshape(n_seq, per).int().cuda()
        self.caches = [bq.KvCache.empty(n_seq * per, self.table, c.kv_type, c.kv_heads, c.head_dim, c.page_tokens)
                       for _ in range(c.layers)]
        self.rope = bq.rope_table(max_len, c.head_dim)
        self.length = torch.zeros(n_seq, dtype=torch.int32, device="cuda")   # tokens cached per sequence
        self.pos = torch.zeros(n_seq, dtype=torch.int32, device="cuda")      # of the decode step's rows
        self.kv_len = torch.zeros(n_seq, dtype=torch.int32, device="cuda")
        self.step = Step(model, self.caches, self.rope, n_seq, self.pos, self.kv_len, max_len, True)
        self.used = [0] * n_seq                                              # of max_len tokens, on the host
        self.tokens = torch.zeros(n_seq, dtype=torch.int32, device="cuda")
        self.u = torch.zeros(n_seq, device="cuda")
        self.gen = torch.Generator(device="cuda").manual_seed(seed)

    def prefill(self, s, prompt, chunk=512):
        """Runs prompt (int32 device tensor) of sequence s in even chunks of at most `chunk` tokens; returns the last
        token's logits [vocab].  (Even, as a few tokens left over would take the decode path, which rounds otherwise.)"""
        import torch
        c, done = self.model.c, 0
        if len(prompt) > self.max_len:
            raise ValueError(f"a prompt of {len(prompt)} tokens: the caches have room for {self.max_len}")
        row = self.table[s: s + 1].contiguous()
        views = [bq.KvCache(k.pages, row, c.kv_type, c.kv_heads, c.head_dim, c.page_tokens) for k in self.caches]
        while done < len(prompt):
            left = len(prompt) - done
            n = -(-left // -(-left // chunk))
            pos = torch.arange(done, done + n, dtype=torch.int32, device="cuda")
            step = Step(self.model, views, self.rope, n, pos, torch.tensor([done + n], dtype=torch.int32, device="cuda"),
                        done + n, False)
            logits = step.run(prompt[done: done + n])
            done += n
        self.length[s] = self.used[s] = len(prompt)
        return logits[-1]

    def set_sampling(self, temperature=0.8, top_k=40, top_p=0.95, min_p=0.0):
        import torch
        n, f = self.n_seq, lambda v, dt=torch.float32: torch.full((self.n_seq,), v, dtype=dt, device="cuda")
        self.rules = dict(temperature=f(temperature), top_k=f(top_k, torch.int32), top_p=f(top_p), min_p=f(min_p))
        self.sampler = bq.Sampler(self.step.logits[:n], self.tokens, self.u, **self.rules)

    def first(self, s, logits):
        """The first token of sequence s from its prompt's last logits."""
        self.u.uniform_(0, 1, generator=self.gen)
        rule = {k: v[s: s + 1] for k, v in self.rules.items()}
        bq.Sampler(logits.reshape(1, -1), self.tokens[s: s + 1], self.u[s: s + 1], **rule).run()

    def decode(self):
        """One more token of every sequence, from self.tokens into self.tokens."""
        if max(self.used) >= self.max_len:
            raise ValueError(f"a sequence has its {self.max_len} tokens: the caches have no room for another")
        self.used = [n + 1 for n in self.used]
        self.pos.copy_(self.length)
        self.length += 1
        self.kv_len.copy_(self.length)
        self.step.run(self.tokens)
        self.u.uniform_(0, 1, generator=self.gen)
        self.sampler.run()
        return self.tokens


def main():
    import time

    import torch
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("batch", 4), ("prompt", 300), ("tokens", 32), ("layers", 2), ("n-embd", 1024), ("q-heads", 8),
                        ("kv-heads", 2), ("n-ff", 2048), ("vocab", 4096), ("window", 0), ("sinks", 0), ("seed", 0)):
        ap.add_argument("--" + name, type=int, default=value)
    ap.add_argument("--kv", choices=("bf16", "q8"), default="bf16")
    a = ap.parse_args()
    if not 1 <= a.batch <= 8:
        ap.error("--batch: 1 to 8 sequences")
    c = Config(n_embd=a.n_embd, q_heads=a.q_heads, kv_heads=a.kv_heads, n_ff=a.n_ff, layers=a.layers, vocab=a.vocab,
               kv_type=a.kv, window=a.window, sinks=a.sinks)
    g = Generator(Model(c, a.seed), a.batch, a.prompt + a.tokens + 1)
    g.set_sampling()
    rng = torch.Generator(device="cuda").manual_seed(a.seed)
    for s in range(a.batch):
        prompt = torch.randint(0, c.vocab, (max(1, a.prompt - 17 * s),), generator=rng, device="cuda", dtype=torch.int32)
        g.first(s, g.prefill(s, prompt))
    g.step.capture()
    out = [g.tokens.clone(), g.decode().clone()]
    torch.cuda.synchronize()
    began = time.perf_counter()
    for _ in range(a.tokens - 1):
        out.append(g.decode().clone())
    torch.cuda.synchronize()
    spent = time.perf_counter() - began
    for s, row in enumerate(torch.stack(out, 1).tolist()):
        print(f"sequence {s}: {row}")
    print(f"{a.tokens - 1} steps of {a.batch} sequences: {spent / max(1, a.tokens - 1) * 1e6:.0f} us a step")


if __name__ == "__main__":
    main()

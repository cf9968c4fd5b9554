"""The serving operators in the decode step (bruce-engine_amd/generate.py):
prompt chunks, then tokens through one captured graph.

* In every step the last layer's attention rows (attn_out) match 64-bit
  attention of that step's own projections (tests/serve_ref.py) over the K and V
  of all tokens so far, which are the projections of earlier steps, normed,
  rotated and rounded as the cache stores them.  Tolerance: as in
  test_gpu_attention.py, plus the storage: the reference's bf16 or q8 rounding of
  a key or value may fall on the other side for a value within fp32 error of
  the boundary, one step of one value (2^-7 of it, or 1/127 of its group's
  largest) in a few thousand; its effect on an output, a weighted mean, stays
  below 2^-7 of sum p |v|, which is added.
* The graph's replays equal an eager run of the same tokens bit for bit, with
  eager work between them, at every length it passes.
* A prompt in one chunk and in several gives the same cache up to that
  rounding, and logits that agree to the q8 activations' resolution.
"""
import pytest
import torch

import serve_ref as R

pytestmark = pytest.mark.gpu


def _config(G, **kw):
    return G.Config(n_embd=512, q_heads=8, kv_heads=2, head_dim=64, n_ff=1024, layers=2, vocab=1024, page_tokens=16, **kw)


class _Watch:
    """What the last layer's append was given, and the attention it should give."""

    def __init__(self, G, c, model, n_seq):
        self.c, self.L = c, model.layers[-1]
        # what the cache stands for, and what the prefill attention's products make of it
        self.k, self.v, self.kh, self.vh = ([[] for _ in range(n_seq)] for _ in range(4))

    def check(self, step, g, seqs, positions, fine):
        c = self.c
        torch.cuda.synchronize()
        rope = g.rope.cpu().double()
        x = [t.cpu().double().reshape(step.rows, -1, c.head_dim) for t in (step.qkv[0], step.qkv[1], step.qkv[3])]
        pos = torch.tensor(positions)
        q, k, v = R.append(*x, pos, rope, c.head_dim, self.L["q_weight"].cpu().double(), self.L["k_weight"].cpu().double(), 1e-6, False)
        if not fine:
            q = R.bf16(q).double() if c.kv_type == "bf16" else R.half_rows(R.bf16(q).float())
        for r, (s, p) in enumerate(zip(seqs, positions)):
            for keep, coarse, t in ((self.k, self.kh, k), (self.v, self.vh, v)):
                t = t[r: r + 1]
                if c.kv_type == "bf16":
                    t = rounded = R.bf16(t).double()
                else:
                    codes, d = R.quant(t.float())
                    t = codes.double() * d.double().repeat_interleave(32, -1)
                    rounded = R.half_keys(codes, d) if coarse is self.kh else R.bf16(t).double()
                assert len(keep[s]) == p
                keep[s].append(t)
                coarse[s].append(rounded)
        got = step.attn_out.cpu().double().reshape(step.rows, c.q_heads, c.head_dim)
        for r, (s, p) in enumerate(zip(seqs, positions)):
            ks, vs = (torch.cat(x[s][: p + 1]) for x in ((self.k, self.v) if fine else (self.kh, self.vh)))
            ref, bound, A = R.attention(q[r: r + 1], ks, vs, [p], c.head_dim ** -0.5, c.window, c.sinks)
            tol = (2.0 ** -16 if fine else 2.0 ** -8) + 2.0 ** -18 * A[..., None] + 2.0 ** -7
            err = (got[r: r + 1] - ref).abs()
            assert (err <= tol * bound).all(), (s, p, (err / (tol * bound)).max())


@pytest.mark.parametrize("kv,window,sinks", [("bf16", 0, 0), ("q8", 0, 0), ("q8", 24, 3)])
def test_prompt_then_tokens(bq, kv, window, sinks):
    import generate as G
    print(f"generate {kv} window {window}", flush=True)
    c = _config(G, kv_type=kv, window=window, sinks=sinks)
    model = G.Model(c, 3)
    n = 3
    g = G.Generator(model, n, 80)
    g.set_sampling(0.9, 30, 0.95, 0.01)
    watch = _Watch(G, c, model, n)
    made = []
    real = G.Step.run

    def run(self, tokens):
        made.append(self)
        return real(self, tokens)
    G.Step.run = run
    try:
        for s, length in enumerate((37, 1, 20)):
            prompt = torch.randint(0, c.vocab, (length,), device="cuda", dtype=torch.int32, generator=g.gen)
            logits = g.prefill(s, prompt, chunk=length)
            watch.check(made[-1], g, [s] * length, list(range(length)), False)
            g.first(s, logits)
    finally:
        G.Step.run = real
    eager_tokens, saved = [], (g.tokens.clone(), g.length.clone(), [k.pages.clone() for k in g.caches], g.gen.get_state())
    rows = []
    for _ in range(6):
        positions = g.length.tolist()
        eager_tokens.append(g.decode().clone())
        watch.check(g.step, g, range(n), positions, True)
        rows.append((g.step.x.clone(), g.step.logits.clone(), g.step.attn_out.clone()))
    # the same tokens through one graph
    g.tokens.copy_(saved[0])
    g.length.copy_(saved[1])
    g.gen.set_state(saved[3])
    for k, p in zip(g.caches, saved[2]):
        k.pages.copy_(p)
    g.step.capture()
    for i in range(6):
        torch.randn(1 << 18, device="cuda").sum()   # unrelated eager work between replays
        torch.cuda.synchronize()
        assert torch.equal(g.decode(), eager_tokens[i]), i
        for a, b in zip(rows[i], (g.step.x, g.step.logits, g.step.attn_out)):
            assert torch.equal(a, b), i
    assert all(((t >= 0) & (t < c.vocab)).all() for t in eager_tokens)


def test_chunks_agree(bq):
    import generate as G
    c = _config(G, kv_type="bf16")
    model = G.Model(c, 4)
    prompt = torch.randint(0, c.vocab, (70,), device="cuda", dtype=torch.int32)
    logits = []
    for chunk in (70, 32):
        g = G.Generator(model, 1, 80)
        logits.append(g.prefill(0, prompt, chunk=chunk).clone())
    # two layers of q8 activations: a code that rounds the other way moves a row by about 3e-4 of its
    # length; the chunks' attention differs by bf16 weights (2^-8 of an output); 2% covers both layers
    a, b = logits
    assert (a - b).norm() <= 0.02 * a.norm()


def test_hook_reports_what_failed(bq):
    """A plan that does not fit the step: the code stays in the plan, later blocks still run."""
    import generate as G
    c = _config(G)
    g = G.Generator(G.Model(c, 5), 1, 32)
    st = g.step.plan.struct
    st.n_blocks = 1           # the second layer's attention block has no entry
    bq.decode_enqueue(g.step.struct)
    with pytest.raises(bq.BqError) as e:
        g.step.plan.check()
    assert e.value.code == bq.BQ_EINVAL
    assert st.status == bq.BQ_OK
    torch.cuda.synchronize()

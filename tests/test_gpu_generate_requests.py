"""A batch of many users' requests through generate.py: a prompt that all sequences
share, an adapter for each, log probabilities of what is drawn, eager and captured.

Two ways to the same logits differ by fp32 or bf16 rounding of the attention (2^-8 of an
output at most) and by codes of the q8 activations that round the other way (3e-4 of a
row's length each, over two layers): 2% of a row of logits, as test_gpu_generate.py has it
for a prompt's chunks.
"""
import ctypes

import pytest
import torch

from test_gpu_generate import _config

pytestmark = pytest.mark.gpu


def _prompts(c, lengths, seed=1):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randint(0, c.vocab, (n,), generator=gen).int().cuda() for n in lengths]


def _close(a, b):
    assert ((a - b).norm(dim=-1) <= 0.02 * a.norm(dim=-1)).all(), ((a - b).norm(dim=-1) / a.norm(dim=-1)).tolist()


def _decode(g, rounds, tokens):
    """The logits of rounds with given tokens."""
    out = []
    for t in tokens[:rounds]:
        g.tokens.copy_(t)
        g.decode()
        out.append(g.step.logits[: g.n_seq].clone())
    return torch.stack(out)


@pytest.mark.parametrize("kv,window,sinks", [("bf16", 0, 0), ("q8", 0, 0), ("bf16", 40, 3)])
@pytest.mark.parametrize("shared", [37, 48, 5])
def test_shared_prompt(bq, kv, window, sinks, shared):
    """A prompt of whole pages, and ones that end inside a page, beside sequences that each hold all of it, run in the
    same pieces (a chunk of few rows takes other matmuls than a long one, and rounds otherwise): the prompts' logits
    are the same bits, the tokens' close."""
    import generate as G
    print(f"shared prompt of {shared}, {kv}, window {window}", flush=True)
    c = _config(G, kv_type=kv, window=window, sinks=sinks)
    model = G.Model(c, 6)
    head, *rest = _prompts(c, (shared, 12, 30, 1, 19))
    n = len(rest)
    a, b = G.Generator(model, n, 120), G.Generator(model, n, 120, shared=True)
    for g in (a, b):
        g.set_sampling()
    b.share(head)
    for s, tail in enumerate(rest):
        a.shared = 0
        a.prefill(s, head)
        a.shared = shared   # go on behind it
        assert torch.equal(a.prefill(s, tail), b.prefill(s, tail))
    assert torch.equal(a.length, b.length) and a.used == b.used
    tokens = [torch.randint(0, c.vocab, (n,), generator=torch.Generator().manual_seed(i)).int().cuda() for i in range(5)]
    _close(_decode(a, 5, tokens), _decode(b, 5, tokens))


def test_share_comes_first(bq):
    import generate as G
    c = _config(G)
    g = G.Generator(G.Model(c, 6, adapters=2), 2, 60, shared=True)
    g.set_sampling()
    head, tail = _prompts(c, (20, 41))
    g.adapter[0] = 1
    with pytest.raises(ValueError):
        g.share(head)
    g.adapter[0] = -1
    g.share(head)
    with pytest.raises(ValueError):
        g.share(head)
    with pytest.raises(ValueError):
        g.prefill(1, tail)


@pytest.mark.parametrize("kv", ["bf16", "q8"])
def test_adapters(bq, kv):
    """Sequences with adapters of their own beside sequences with none: each as if it were alone."""
    import generate as G
    c = _config(G, kv_type=kv)
    model = G.Model(c, 7, adapters=3, rank=16)
    prompts = _prompts(c, (21, 9, 33, 14), 2)
    slots = [2, -1, 0, 2]
    tokens = [torch.randint(0, c.vocab, (4,), generator=torch.Generator().manual_seed(10 + i)).int().cuda() for i in range(4)]
    g = G.Generator(model, 4, 60)
    g.set_sampling()
    g.adapter.copy_(torch.tensor(slots))
    first = [g.prefill(s, p).clone() for s, p in enumerate(prompts)]
    got = _decode(g, 4, tokens)
    for s, (p, slot) in enumerate(zip(prompts, slots)):
        one = G.Generator(model, 1, 60)
        one.set_sampling()
        one.adapter.fill_(slot)
        _close(one.prefill(0, p), first[s])
        _close(_decode(one, 4, [t[s: s + 1] for t in tokens])[:, 0], got[:, s])
        if slot >= 0:  # and an adapter changes what the base model says
            base = G.Generator(model, 1, 60)
            base.set_sampling()
            other = base.prefill(0, p)
            assert (other - first[s]).norm() > 0.02 * other.norm()


def test_adapters_that_add_nothing(bq):
    """An adapter of zeros is the base model, bit for bit."""
    import generate as G
    c = _config(G)
    model = G.Model(c, 8, adapters=2, rank=8)
    for layer in model.lora:
        for parts in layer.values():
            for _, b in parts:
                b[1].zero_()
    prompt, = _prompts(c, (25,), 3)
    out = []
    for slot in (-1, 1):
        g = G.Generator(model, 1, 40)
        g.set_sampling()
        g.adapter.fill_(slot)
        out.append((g.prefill(0, prompt).clone(), _decode(g, 2, [prompt[:1], prompt[1:2]])))
    assert all(torch.equal(a, b) for a, b in zip(*out))


@pytest.mark.parametrize("kv", ["bf16", "q8"])
def test_all_together_captured(bq, kv):
    """A shared prompt, adapters, sampling and log probabilities: the captured step's replays equal the eager ones with
    other work between, and what LogProbs says is what the logits say."""
    import generate as G
    c = _config(G, kv_type=kv)
    g = G.Generator(G.Model(c, 9, adapters=3, rank=24), 5, 100, shared=True)
    g.set_sampling(0.9, 30, 0.95, 0.0, logprobs=4)
    head, *rest = _prompts(c, (35, 7, 20, 3, 11, 16), 4)
    g.share(head)
    g.adapter.copy_(torch.tensor([0, 2, -1, 1, 2]))
    for s, tail in enumerate(rest):
        g.first(s, g.prefill(s, tail))
    state = g.tokens.clone(), g.length.clone(), list(g.used), [k.pages.clone() for k in g.caches], g.gen.get_state()
    eager = []
    for _ in range(5):
        t = g.decode().clone()
        eager.append((t, g.step.logits.clone(), {k: v.clone() for k, v in g.logprobs.items()}))
        z = eager[-1][1][:5].double() / g.rules["temperature"].double()[:, None]
        lp = torch.log_softmax(z, 1)
        order = torch.argsort(z, dim=1, descending=True, stable=True)
        got = eager[-1][2]
        # fp32 against 64 bits: 2^-20 of exponents below 64
        assert (got["logprob"].double() - lp.gather(1, t.long()[:, None])[:, 0]).abs().max() <= 2.0 ** -14
        assert (got["entropy"].double() + (lp.exp() * lp).sum(1)).abs().max() <= 2.0 ** -14
        assert torch.equal(got["top_tokens"].long(), order[:, :4])
        assert torch.equal(got["rank"].long(), (order == t.long()[:, None]).int().argmax(1))
    g.tokens.copy_(state[0])
    g.length.copy_(state[1])
    g.used = state[2]
    g.gen.set_state(state[4])
    for k, pages in zip(g.caches, state[3]):
        k.pages.copy_(pages)
    g.step.capture()
    for t, logits, lp in eager:
        torch.randn(1 << 18, device="cuda").sum()
        torch.cuda.synchronize()
        assert torch.equal(g.decode(), t) and torch.equal(g.step.logits, logits)
        assert all(torch.equal(g.logprobs[k], v) for k, v in lp.items())


def test_hook_reports_what_failed(bq):
    """An adapter call that is refused: the code stays in the plan, the step goes on."""
    import generate as G
    c = _config(G)
    g = G.Generator(G.Model(c, 5, adapters=2), 2, 32)
    st = g.step.adapters.struct
    st.blocks[1].proj[bq.PROJ_DOWN].contents.work_bytes = 0
    bq.decode_enqueue(g.step.struct)
    with pytest.raises(bq.BqError) as e:
        g.step.adapters.check()
    assert e.value.code == bq.BQ_EINVAL and st.status == bq.BQ_OK
    torch.cuda.synchronize()

"""What generate.py reserves, and where it ends: one workspace for the layers of a
step, sized by the tokens that are there, and an error where the caches are full."""
import pytest
import torch

from test_gpu_generate import _config

pytestmark = pytest.mark.gpu


def _steps(G, f):
    """The steps that f() runs."""
    made, real = [], G.Step.run

    def run(self, tokens):
        made.append(self)
        return real(self, tokens)
    G.Step.run = run
    try:
        f()
    finally:
        G.Step.run = real
    return made


def _works(step):
    return [(b.attn.contents.work, b.attn.contents.work_bytes) for b in step.plan._blocks if b.attn]


def test_layers_share_a_workspace_of_the_tokens_size(bq):
    import generate as G
    c = _config(G, kv_type="q8")
    model = G.Model(c, 5)
    prompt = torch.randint(0, c.vocab, (520,), generator=torch.Generator().manual_seed(1)).int().cuda()
    got = []
    for room in (600, 9000):
        g = G.Generator(model, 2, room)
        g.set_sampling()
        out = []
        step, = _steps(G, lambda: out.append(g.prefill(0, prompt, chunk=520)))
        works = _works(step)
        assert len(works) == c.layers and len(set(works)) == 1 and works[0][1] > 0
        assert len(set(_works(g.step))) == 1
        got.append((works[0][1], out[0].clone()))
    # the same tokens: the same workspace and the same logits, whatever the caches have room for
    assert got[0][0] == got[1][0]
    assert torch.equal(got[0][1], got[1][1])


def test_full_caches_are_an_error(bq):
    import generate as G
    c = _config(G)
    g = G.Generator(G.Model(c, 6), 2, 20)
    g.set_sampling()
    gen = torch.Generator().manual_seed(2)
    with pytest.raises(ValueError):
        g.prefill(0, torch.randint(0, c.vocab, (21,), generator=gen).int().cuda())
    for s, n in ((0, 5), (1, 18)):
        g.first(s, g.prefill(s, torch.randint(0, c.vocab, (n,), generator=gen).int().cuda()))
    g.decode()
    g.decode()
    tokens, length = g.tokens.clone(), g.length.tolist()
    with pytest.raises(ValueError):
        g.decode()
    assert g.length.tolist() == length == [7, 20] and torch.equal(g.tokens, tokens)

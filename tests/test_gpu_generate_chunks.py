"""A prompt cut in different ways gives the same logits, chunks of few rows (which take other matmul kernels)
among them.

Tolerance, of the logits' norm: per layer the attention rounds queries, weights and values or outputs to bf16, 2^-8
of an output each; a q8 activation that rounds the other way moves a row by 3e-4 of its length, in each of a layer's
four matmuls: 2 * (3 * 2^-8 + 4 * 3e-4) = 2.6%.  Chunks of more than 8 rows take the same kernels, row by row, and
round alike but for such codes: 2 * 4 * 3e-4.
"""
import pytest
import torch

from test_gpu_generate import _config

pytestmark = pytest.mark.gpu


def _logits(bq, G, model, prompt, sizes):
    """The last token's logits after the prompt in chunks of these sizes."""
    c, g = model.c, G.Generator(model, 1, 80)
    done = 0
    for n in sizes:
        pos = torch.arange(done, done + n, dtype=torch.int32, device="cuda")
        step = G.Step(model, g.caches, g.rope, n, pos, torch.tensor([done + n], dtype=torch.int32, device="cuda"), done + n, False)
        out = step.run(prompt[done: done + n])
        done += n
    assert done == len(prompt)
    return out[-1].clone()


@pytest.mark.parametrize("kv", ["bf16", "q8"])
@pytest.mark.parametrize("seed", [11, 12, 13])
def test_cuts_of_a_prompt_agree(bq, kv, seed):
    import generate as G
    c = _config(G, kv_type=kv)
    model = G.Model(c, seed)
    prompt = torch.randint(0, c.vocab, (70,), generator=torch.Generator().manual_seed(seed)).int().cuda()
    whole = _logits(bq, G, model, prompt, (70,))
    assert torch.equal(whole, G.Generator(model, 1, 80).prefill(0, prompt, chunk=70))
    for sizes in ((35, 35), (64, 6), (6, 64), (1, 69), (62, 8), (23, 23, 24)):
        off = ((_logits(bq, G, model, prompt, sizes) - whole).norm() / whole.norm()).item()
        print(f"  {kv} seed {seed} {sizes}: {off:.2e}", flush=True)
        assert off <= 2 * ((3 * 2.0 ** -8 if min(sizes) <= 8 else 0) + 4 * 3e-4), sizes

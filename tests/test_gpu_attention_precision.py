"""How exact attention is, term by term, and against the definition (reference: tests/serve_ref.py).

test_decode_terms: each token's value has one dim of its own, so an output value is one softmax weight, and each
score is one product of an fp32 query value and a key value, |score| <= 1.  An output may be off, relatively, by
  the exponent's argument |x| <= 1.5: scale log2(e), product and x - m rounded to 2^-24 each: 2^-22 of the weight,
    and as much of the sum of the weights;
  2^-23 for the exponential, each way; the sum of 64 weights over 8 in a lane, 4 lane groups and 4 waves: 14
    roundings of 2^-24; the division and the product with its reciprocal 2^-23:  together below 2^-19.
What a part of an operand that got lost would cost is more: the third bf16 part of a query or a weight 2^-17 (16 bits
left), the second of a weight over q8 2^-8, of an fp16 query 2^-11.  Over a bf16 cache 2^-19 is the tolerance.  Over
q8 a query is two fp16 parts (2^-22 of its largest value, which it is here) and a weight times a value's scale two
bf16 parts, 2^-17 more of each term: 2^-16.

test_prefill_against_definition: queries are rounded to bf16 (2^-8 of a value), over q8 to fp16 (2^-11), there with
the keys (a scale and a product, 2^-11 each).  With A = scale sum |q_i k_i| a score moves by r A, r = 2^-8 or
3 * 2^-11, a weight and the sum of the weights by (e^(r A) - 1) of itself each; weights and values bf16 and a bf16
output as in test_gpu_attention.py.
"""
import numpy as np
import pytest
import torch

import serve_ref as R
from test_gpu_attention import _normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [2, 17, 64])
@pytest.mark.parametrize("kv", ["bf16", "q8"])
@pytest.mark.parametrize("D,rows", [(64, 1), (128, 1), (128, 4), (256, 1)])
def test_decode_terms(bq, kv, D, rows, T):
    H, G, P = 1, 8, 32
    rng = np.random.default_rng(T + D)
    pages = R.Pages(kv, H, D, P, 1, (T + P - 1) // P, 3)
    k, v = torch.zeros((T, H, D)), torch.zeros((T, H, D))
    # a key group of one value: its q8 code is 127 and its scale carries the size, exact in fp32
    k[:, 0, 0] = R.bf16(torch.from_numpy(rng.uniform(-1, 1, T).astype(np.float32)) * 0.98).float()
    v[torch.arange(T), 0, torch.arange(T) % D] = 1.0
    pages.put(0, k, v)
    q = torch.zeros((rows, G, D))
    q[:, :, 0] = torch.from_numpy(rng.uniform(0.5, 1, (rows, G)).astype(np.float32))  # all 24 bits
    out = torch.empty((rows, G * D), device="cuda")
    bq.Attention(pages.cache(bq), q.reshape(rows, -1).cuda(), out, torch.tensor([T], dtype=torch.int32, device="cuda"), scale=1.0).decode()
    got = out.cpu().double().reshape(rows, G, D)
    ref, _, _ = R.attention(q.double(), pages.k[0], pages.v[0], torch.arange(T - rows, T), 1.0)
    assert (got[ref == 0] == 0).all()
    err = ((got - ref).abs() / ref.abs().clamp(min=1e-300))[ref != 0].max().item()
    tol = 2.0 ** -19 if kv == "bf16" else 2.0 ** -16
    print(f"  {kv} D {D} {rows} rows {T} tokens: worst relative error 2^{np.log2(max(err, 1e-30)):.2f}", flush=True)
    assert err <= tol


@pytest.mark.parametrize("kv", ["bf16", "q8"])
@pytest.mark.parametrize("qt,ot", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")])
@pytest.mark.parametrize("D,Hq,H,rows,past", [(64, 8, 2, 90, 40), (128, 4, 1, 33, 300), (256, 8, 1, 270, 0)])
def test_prefill_against_definition(bq, kv, qt, ot, D, Hq, H, rows, past):
    dt = {"f32": torch.float32, "bf16": torch.bfloat16}
    T, P = rows + past, 64
    pages = R.Pages(kv, H, D, P, 1, (T + P - 1) // P, 5)
    pages.put(0, _normal(D, T, H, D), _normal(D + 1, T, H, D))
    q = (_normal(D + 2, rows, Hq * D) * 0.5).to(dt[qt])
    for work in ("auto", None):
        out = torch.empty((rows, Hq * D), dtype=dt[ot], device="cuda")
        bq.Attention(pages.cache(bq), q.cuda(), out, torch.tensor([T], dtype=torch.int32, device="cuda"), work=work,
                     row0=torch.tensor([0, rows], dtype=torch.int32, device="cuda"), max_rows=rows).prefill()
        got = out.cpu().double().reshape(rows, Hq, D)
        ref, bound, A = R.attention(q.double().reshape(rows, Hq, D), pages.k[0], pages.v[0], torch.arange(past, T), D ** -0.5)
        r = 3 * 2.0 ** -11 if kv == "q8" else 2.0 ** -8 if qt == "f32" else 0.0
        tol = 2 * torch.expm1(r * A) + 2.0 ** -7 * (1 + 2.0 ** -6) + 2.0 ** -18 * A
        if kv == "q8":
            tol = tol + 2.0 ** -8  # values rounded to bf16
        ratio = ((got - ref).abs() / (tol[..., None] * bound).clamp(min=1e-30)).max().item()
        off = ((got - ref).norm() / ref.norm()).item()
        print(f"  {kv} {qt}->{ot} D {D} {rows} rows of {T}, work {work}: worst error / tolerance {ratio:.3f}, norm {off:.2e}", flush=True)
        assert torch.isfinite(got).all() and ratio <= 1

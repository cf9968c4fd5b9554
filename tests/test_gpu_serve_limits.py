"""What the serving operators refuse because an index could not hold it."""
import ctypes

import pytest
import torch

import serve_ref as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("P", [16, 32, 64, 128, 256])
def test_table_rows_that_pass_32_bits(bq, P):
    """A tile that ends past token 2^31 - 1 would have a negative end; shorter rows are served."""
    L, D = bq.load(), 64
    cache = R.Pages("bf16", 1, D, P, 1, 1, 3).cache(bq)
    q = torch.zeros((1, D), device="cuda")
    out = torch.full((1, D), 7.0, device="cuda")
    ok = bq.Attention(cache, q, out, torch.zeros(1, dtype=torch.int32, device="cuda"), work=None)
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    most = (2 ** 31 - 128) // P
    for pages, code in ((most + 1, bq.BQ_UNSUPPORTED), (most, bq.BQ_OK)):
        c, a = bq.KvCacheStruct.from_buffer_copy(cache.struct), bq.AttnArgs.from_buffer_copy(ok.struct)
        c.max_pages, a.max_len = pages, 2 ** 31 - 1
        for f in (L.bq_attn_decode, L.bq_attn_prefill):   # (length 0: no entry of the table is read)
            assert f(ctypes.byref(c), ctypes.byref(a), bq._stream()) == code, (f, pages)
        if code != bq.BQ_OK:
            assert L.bq_kv_read(ctypes.byref(c), None, pos.data_ptr(), 1, None, None, bq._stream()) == code
            torch.cuda.synchronize()
            assert (out == 7).all()
    torch.cuda.synchronize()
    assert (out == 0).all()

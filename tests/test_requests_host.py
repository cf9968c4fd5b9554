"""CPU checks of the operators for batches of many users' requests: the ctypes mirrors of
their structures, the host-only size functions, and the binding on tensors of the wrong
place, type or shape (stand-ins for device tensors; nothing is launched)."""
import contextlib
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

import bq
from test_abi import ROOT, header_fields
from test_serve_binding import Fake

STRUCTS = [("bq_attn_prefix", "AttnPrefix"), ("bq_attn_block", "AttnBlock"), ("bq_lora_part", "LoraPart"), ("bq_lora_args", "LoraArgs"),
           ("bq_lora_block", "LoraBlock"), ("bq_lora_plan", "LoraPlanStruct"), ("bq_logprobs_args", "LogprobsArgs"),
           ("bq_decode_step", "DecodeStep")]


def test_ctypes_structs_match_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    src = ['#include <stddef.h>', '#include <stdio.h>', '#include "bq.h"', 'int main(void) {']
    for cname, pyname in STRUCTS:
        src.append('printf("%s size %%zu\\n", sizeof(%s));' % (cname, cname))
        for f, _ in getattr(bq, pyname)._fields_:
            src.append('printf("%s %s %%zu\\n", offsetof(%s, %s));' % (cname, f, cname, f))
    src.append('printf("max top %d\\nmax rows %d\\nmax rank %d\\nparts %d\\nprojections %d %d %d %d %d\\n", BQ_MAX_TOP, BQ_MAX_LORA_ROWS, BQ_MAX_RANK, BQ_MAX_PARTS, BQ_PROJ_QKV, '
               'BQ_PROJ_O, BQ_PROJ_GATE_UP, BQ_PROJ_DOWN, BQ_N_PROJ);')
    src.append("return 0; }")
    (tmp_path / "off.c").write_text("\n".join(src))
    exe = tmp_path / "off"
    subprocess.run([cc, "-I", os.path.join(ROOT, "include"), str(tmp_path / "off.c"), "-o", str(exe)], check=True)
    got = dict(l.rsplit(" ", 1) for l in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for cname, pyname in STRUCTS:
        S = getattr(bq, pyname)
        assert int(got[f"{cname} size"]) == ctypes.sizeof(S), cname
        for f, _ in S._fields_:
            assert int(got[f"{cname} {f}"]) == getattr(S, f).offset, (cname, f)
    assert got["max top"] == "64" and got["max rows"] == str(1 << 20) and got["max rank"] == "256" and got["parts"] == "4"
    assert [bq.PROJ_QKV, bq.PROJ_O, bq.PROJ_GATE_UP, bq.PROJ_DOWN] == [0, 1, 2, 3] and got["projections 0 1 2 3"] == "4"
    for cname, pyname in STRUCTS[:2] + STRUCTS[5:]:
        assert [f[0] for f in getattr(bq, pyname)._fields_][: len(header_fields(cname))] == header_fields(cname), cname


def test_workspace_bytes():
    L = bq.load()
    f = L.bq_logprobs_workspace_bytes
    assert 0 < f(1, 1, 0) <= f(1, 131072, 0) < f(1, 131072, 5) <= f(1, 131072, 64) and f(64, 131072, 20) == 64 * f(1, 131072, 20)
    for bad in ((0, 100, 1), (1, 0, 1), (1, (1 << 20) + 1, 1), (1, 100, 65), (1, 100, -1)):
        assert f(*bad) == 0, bad
    g = L.bq_lora_workspace_bytes
    # t is there at least once, and no piece is smaller than it
    for rows in (1, 16, 255, 256, 257, 8192):
        for rank in (8, 16, 256):
            for parts in (1, 2, 3, 4):
                n = g(rows, rank, parts)
                assert n % (4 * rows * rank * parts) == 0 and 1 <= n // (4 * rows * rank * parts) <= 8, (rows, rank, parts)
    for bad in ((0, 8, 1), (1, 0, 1), (1, 264, 1), (1, 8, 0), (1, 8, 5)):
        assert g(*bad) == 0, bad


I, F, H, B = torch.int32, torch.float32, torch.bfloat16, torch.int8
D, P = 64, 16


def _cache():
    return bq.KvCache(Fake(torch.uint8, 4, bq.kv_page_bytes("bf16", 1, D, P)), Fake(I, 2, 2), "bf16", 1, D, P)


ARGS = {"shared": dict(q=(F, 2, D), out=(F, 2, D), kv_len=(I, 2), group0=(I, 2), prefix_len=(I, 1), work=(F, 100)),
        "lora": dict(x=(F, 3, 64), adapter=(I, 3), a=(H, 2, 8, 64), b=(H, 2, 32, 8), y=(F, 3, 32), base=(F, 3, 32), scale=(F, 2),
                     work=(torch.uint8, 1 << 20)),
        "lora_q8": dict(x=(B, 3, 64), xd=(F, 3, 2), adapter=(I, 3), a=(H, 2, 8, 64), b=(H, 2, 32, 8), y=(F, 3, 32), base=(F, 3, 32)),
        "logprobs": dict(logits=(F, 2, 100), tokens=(I, 2), logprob=(F, 2), rank=(I, 2), entropy=(F, 2), top_tokens=(I, 2, 5),
                         top_logprobs=(F, 2, 5), temperature=(F, 2), work=(torch.uint8, 1 << 20))}


def _make(op, name=None, dtype=None, shape=None, **how):
    """The operator's object over tensors of device 0, `name` made otherwise."""
    a = {n: Fake(dtype if n == name and dtype else t[0], *(shape if n == name and shape else t[1:]), **(how if n == name else {}))
         for n, t in ARGS[op].items()}
    if op == "shared":
        return bq.SharedAttention(_cache(), **a)
    if op == "logprobs":
        return bq.LogProbs(**a)
    part = [(a["a"], a["b"], a["y"], a["base"])]
    return bq.Lora((a["x"], a["xd"]) if "xd" in a else a["x"], a["adapter"], part, scale=a.get("scale"), work=a.get("work"))


@pytest.mark.parametrize("op", list(ARGS))
def test_tensors_of_another_device(op):
    """Each tensor on a second GPU, and on the host: refused before anything is called."""
    for name in ARGS[op]:
        for how in (dict(index=1), dict(cuda=False)):
            with pytest.raises(ValueError):
                _make(op, name, **how)


@pytest.mark.parametrize("op,name,dtype,shape", [
    ("shared", "group0", None, (3,)), ("shared", "prefix_len", torch.int64, None), ("shared", "kv_len", None, (1,)), ("shared", "out", None, (2, 2 * D)),
    ("shared", "q", None, (2, 60)), ("lora", "adapter", torch.int64, None), ("lora", "adapter", None, (2,)), ("lora", "a", F, None),
    ("lora", "a", None, (2, 8, 32)), ("lora", "b", None, (2, 32, 16)), ("lora", "y", H, None), ("lora", "y", None, (4, 32)), ("lora", "base", None, (3, 48)),
    ("lora", "scale", None, (3,)), ("lora_q8", "xd", None, (3, 1)), ("lora_q8", "x", I, None), ("logprobs", "tokens", torch.int64, None),
    ("logprobs", "rank", F, None), ("logprobs", "top_logprobs", None, (2, 4)), ("logprobs", "entropy", None, (3,)), ("logprobs", "temperature", None, (1,))])
def test_types_and_shapes(op, name, dtype, shape):
    with pytest.raises((ValueError, TypeError)):
        _make(op, name, dtype, shape)


def test_types_that_are_not_taken():
    with pytest.raises(TypeError):
        _make("logprobs", "logits", H)
    with pytest.raises(TypeError):
        _make("lora", "x", torch.float16)
    x, ad = Fake(F, 3, 64), Fake(I, 3)
    part = (Fake(H, 2, 8, 64), Fake(H, 2, 32, 8), Fake(F, 3, 32))
    with pytest.raises(ValueError):
        bq.Lora(x, ad, [part] * 5)


def test_workspaces_that_are_not_there():
    for op in ("shared", "lora", "logprobs"):
        with pytest.raises(ValueError):
            _make(op, "work", contiguous=False)


@pytest.mark.parametrize("current", [0, 1])
def test_calls_go_to_the_tensors_device(monkeypatch, current):
    """The launch, not only the stream, is the tensors' device's, whichever is current; the current one comes back."""
    now, seen = [current], []

    @contextlib.contextmanager
    def device(d):
        before, now[0] = now[0], d
        yield
        now[0] = before
    bq._bind_device()
    monkeypatch.setattr(bq, "_current", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(bq, "_raw_stream", lambda d: 1000 + d)
    for op in ("shared", "lora", "logprobs"):
        obj = _make(op)
        obj._run = lambda *a: seen.append((now[0], a[-1])) or 0
        obj.run()
    assert seen == [(0, 1000)] * 3 and now == [current]


def test_plans():
    """What the plans' structures hold of the operators' arguments."""
    lora = _make("lora")
    plan = bq.LoraPlan([{bq.PROJ_O: lora}, None, {}])
    assert plan.struct.n_blocks == 3 and ctypes.addressof(plan._blocks[0].proj[bq.PROJ_O].contents) == ctypes.addressof(lora.struct)
    assert not plan._blocks[0].proj[bq.PROJ_QKV] and not any(plan._blocks[1].proj) and not any(plan._blocks[2].proj)
    plan.struct.status = bq.BQ_EINVAL
    with pytest.raises(bq.BqError):
        plan.check()
    assert plan.check() == bq.BQ_OK
    step = plan.install(bq.DecodeStep())
    assert ctypes.cast(step.projected, ctypes.c_void_p).value == ctypes.cast(bq.load().bq_lora_hook, ctypes.c_void_p).value
    assert step.projected_user == ctypes.addressof(plan.struct)

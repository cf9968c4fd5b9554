"""CPU checks of the serving operators: the ctypes mirrors of their structures,
the host-only size functions, and the direct-to-LDS copies of the prefill
attention, which write m0 in inline asm: as in the prefill GEMMs (see
test_isa_m0.py) nothing else in those kernels may use m0."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest

from test_abi import ROOT, header_fields
from test_isa_m0 import IMPLICIT_M0, OBJDUMP

STRUCTS = [("bq_kv_cache", "KvCacheStruct"), ("bq_append_args", "AppendArgs"), ("bq_attn_args", "AttnArgs"),
           ("bq_attn_block", "AttnBlock"), ("bq_attn_plan", "AttnPlanStruct")]


def test_ctypes_structs_match_header(tmp_path):
    import bq
    for cname, pyname in STRUCTS:
        assert [f[0] for f in getattr(bq, pyname)._fields_] == header_fields(cname), cname
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    src = ['#include <stddef.h>', '#include <stdio.h>', '#include "bq.h"', 'int main(void) {']
    for cname, _ in STRUCTS:
        src.append('printf("%s size %%zu\\n", sizeof(%s));' % (cname, cname))
        for f in header_fields(cname):
            src.append('printf("%s %s %%zu\\n", offsetof(%s, %s));' % (cname, f, cname, f))
    src.append("return 0; }")
    (tmp_path / "off.c").write_text("\n".join(src))
    exe = tmp_path / "off"
    subprocess.run([cc, "-I", os.path.join(ROOT, "include"), str(tmp_path / "off.c"), "-o", str(exe)], check=True)
    got = dict(l.rsplit(" ", 1) for l in subprocess.run([str(exe)], capture_output=True, text=True,
                                                        check=True).stdout.splitlines())
    for cname, pyname in STRUCTS:
        S = getattr(bq, pyname)
        assert int(got[f"{cname} size"]) == ctypes.sizeof(S), cname
        for f, _ in S._fields_:
            assert int(got[f"{cname} {f}"]) == getattr(S, f).offset, (cname, f)


def test_page_bytes():
    import bq
    assert bq.kv_page_bytes("bf16", 4, 128, 64) == 4 * 64 * 128 * 2 * 2
    assert bq.kv_page_bytes("q8", 8, 64, 16) == 8 * 16 * 64 * 2 * (1 + 2 / 32)
    for bad in ((30, 4, 96, 64), (30, 4, 128, 24), (30, 0, 128, 64), (13, 4, 128, 64), (30, 4, 128, 512)):
        assert bq.load().bq_kv_page_bytes(*bad) == 0, bad
    with pytest.raises(bq.BqError):
        bq.kv_page_bytes("q8", 4, 80, 64)


def test_sample_workspace_bytes():
    import bq
    f = bq.load().bq_sample_workspace_bytes
    assert f(0, 100) == 0 and f(1, 0) == 0 and f(1, (1 << 20) + 1) == 0
    assert 0 < f(1, 1) <= f(1, 131072) and f(64, 131072) == 64 * f(1, 131072)


def test_prefill_attention_m0(tmp_path):
    src = os.path.join(ROOT, "bruce-engine_amd", "_build", "bq_attn_prefill.o")
    if not (os.path.exists(src) and os.path.exists(OBJDUMP)):
        pytest.skip("needs the built bq_attn_prefill.o (bruce-engine_amd/build.py) and llvm-objdump")
    obj = tmp_path / "o.o"
    shutil.copy(src, obj)
    subprocess.run([OBJDUMP, "--offloading", str(obj)], check=True, capture_output=True, cwd=tmp_path)
    co = [f for f in os.listdir(tmp_path) if f.endswith("gfx950")]
    assert co
    text = subprocess.run([OBJDUMP, "-d", "--mcpu=gfx950", str(tmp_path / co[0])], check=True, capture_output=True,
                          text=True).stdout
    insts = [l.split("//")[0].strip() for l in text.splitlines() if l.startswith("\t")]
    writes = 0
    for j, ins in enumerate(insts):
        assert not IMPLICIT_M0.search(ins), ins
        if re.search(r"\bm0\b", ins):
            assert ins.startswith("s_mov_b32 m0,"), ins
            n = j + 1
            while insts[n].startswith("s_nop"):
                n += 1
            assert insts[n].startswith("global_load_lds_dwordx4"), (ins, insts[n])
            writes += 1
        if ins.startswith("global_load_lds"):
            p = j - 1
            while insts[p].startswith("s_nop"):
                p -= 1
            assert insts[p].startswith("s_mov_b32 m0,"), (ins, insts[p])
    assert writes > 0
    # packed fp32 arithmetic stays off
    assert not re.search(r"v_pk_(add|mul|fma)_f32", text)

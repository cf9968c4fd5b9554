"""What the compiler must not pass over in silence (CPU: hipcc only)."""
import os
import subprocess

import pytest

from test_abi import ROOT

CSRC = os.path.join(ROOT, "bruce-engine_amd", "csrc")


def _hipcc(path):
    import build
    if not os.path.exists(build.HIPCC):
        pytest.skip("needs hipcc")
    r = subprocess.run([build.HIPCC] + build.CFLAGS + ["-fsyntax-only", path], capture_output=True, text=True)
    return r.returncode, r.stderr


def test_an_unknown_attribute_ends_the_build(tmp_path):
    """16-byte LDS accesses rest on the alignment that an array is declared with: an attribute spelt wrongly is
    ignored by default, and the array keeps its type's."""
    src = tmp_path / "a.hip"
    body = '#include <hip/hip_runtime.h>\n__global__ void k(float* p) {\n  __shared__ __attribute__((%s)) float s[64];\n' \
           '  s[threadIdx.x] = p[threadIdx.x];\n  __syncthreads();\n  p[threadIdx.x] = s[63 - threadIdx.x];\n}\n'
    src.write_text(body % "aligned(16)")
    assert _hipcc(str(src))[0] == 0
    src.write_text(body % "aligned16")
    code, err = _hipcc(str(src))
    assert code != 0 and "unknown attribute" in err, err


@pytest.mark.parametrize("name", ["bq_attn.hip", "bq_attn_prefill.hip", "bq_kv.hip", "bq_sample.hip"])
def test_no_attribute_is_ignored(name):
    code, err = _hipcc(os.path.join(CSRC, name))
    assert code == 0 and "ignored" not in err, err

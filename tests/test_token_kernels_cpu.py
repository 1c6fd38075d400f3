"""CPU: the compiled token kernels (layer norm, dropout, attention): no scratch memory, no packed fp32 arithmetic, products on the matrix cores."""
import os
import re
import subprocess
import tempfile
from concurrent.futures import ThreadPoolExecutor

import pytest

from pdae_amd import build as B

SRCS = ["layernorm.hip", "dropout.hip", "mha_fwd.hip", "mha_bwd.hip"]


def compiled(src):
    """({kernel: scratch bytes a lane}, device assembly) of csrc/<src>, built as the library is."""
    with tempfile.TemporaryDirectory() as td:
        cmd = [B.HIPCC] + B.FLAGS + B.EXTRA_FLAGS[src] + ["-Rpass-analysis=kernel-resource-usage", "--save-temps=obj", "-c", os.path.join(B.CSRC, src), "-o",
                                                          os.path.join(td, "o.o")]
        r = subprocess.run(cmd, capture_output=True, text=True, cwd=td)
        assert r.returncode == 0, r.stderr[-2000:]
        asm = "".join(open(os.path.join(td, f)).read() for f in os.listdir(td) if f.endswith(".s") and "amdgcn" in f)
    names = re.findall(r"Function Name: (\S+)", r.stderr)
    scratch = re.findall(r"ScratchSize \[bytes/lane\]: (\d+)", r.stderr)
    assert names and len(names) == len(scratch)
    return dict(zip(names, map(int, scratch))), asm


@pytest.fixture(scope="module")
def built():
    with ThreadPoolExecutor(max_workers=4) as ex:
        return dict(zip(SRCS, ex.map(compiled, SRCS)))


@pytest.mark.timeout(900)
def test_token_kernels_use_no_scratch_memory(built):
    bad = {k: n for t, _ in built.values() for k, n in t.items() if n}
    assert not bad, bad


def test_token_kernels_hold_no_packed_fp32_arithmetic(built):
    for src, (_, asm) in built.items():
        assert "s_endpgm" in asm
        assert not re.findall(r"\bv_pk_(?:add|mul|fma)_f32\b", asm), src


def test_attention_products_run_on_the_matrix_cores(built):
    for src in ("mha_fwd.hip", "mha_bwd.hip"):
        table, asm = built[src]
        for name in table:
            body = asm.split("\n%s:" % name, 1)[1].split("\n.Lfunc_end", 1)[0]
            n = len(re.findall(r"v_mfma_f32_32x32x16_bf16", body))
            assert (n == 0) == ("join" in name), (name, n)

"""Static checks on the gfx950 assembly hipcc generates for the kernels of 4-bit weights and of the mixture-of-experts layer (no GPU needed).

Their rings are filled by direct loads whose asm statements leave M0 changed, and counted waits tell that they have arrived.  Neither is known to the compiler, so:

  * no instruction that the compiler generated names M0, and each direct load stands right behind the setting of M0;
  * the loops wait with the counts that the kernels are written for: every stream and tile kernel has a wait for a number of loads that is not 0;
  * nothing is spilled to scratch memory: its loads would be counted among the others;
  * no packed fp32 instruction.
"""
import os
import re
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from test_kernel_asm import CSRC, FLAGS, HIPCC, _compiler_generated, _kernels

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not installed")


@pytest.fixture(scope="module")
def asm_files(tmp_path_factory):
    outdir = str(tmp_path_factory.mktemp("w4_asm"))

    def compile_one(src):
        out = os.path.join(outdir, src.replace(".hip", ".s"))
        r = subprocess.run([HIPCC] + FLAGS + [os.path.join(CSRC, src), "-o", out], capture_output=True, text=True)
        assert r.returncode == 0, r.stderr[-3000:]
        return out

    with ThreadPoolExecutor(2) as pool:
        return list(pool.map(compile_one, ["w4.hip", "moe.hip"]))


def _rings(asm_files):
    for path in asm_files:
        for name, body in _kernels(path).items():
            if any(t.startswith("global_load_lds") for t in body):
                yield name, body


def test_m0_belongs_to_the_direct_loads(asm_files):
    for path in asm_files:
        for name, body in _compiler_generated(path).items():
            bad = [t for t in body if re.search(r"\bm0\b", t) or t.startswith("global_load_lds")]
            assert not bad, f"{name}: {bad[:3]}"
    checked = 0
    for name, body in _rings(asm_files):
        for i, t in enumerate(body):
            if t.startswith("global_load_lds"):
                assert body[i - 2].startswith("s_mov_b32 m0, s") and body[i - 1] == "s_nop 0", f"{name}: {body[i - 2:i + 1]}"
                checked += 1
    assert checked > 1000


def test_rings_wait_for_counted_loads(asm_files):
    rings = list(_rings(asm_files))
    for name, body in rings:
        assert any(re.match(r"s_waitcnt vmcnt\([1-9]\d*\)( lgkmcnt\(0\))?$", t) for t in body), name
    # gemm_w4: streams of 1, 4, 16 and 32 columns and tiles; the layer's two products for 1, 4 and 16 columns; each in both types
    for part in ("gemm_w4_stream_kernel", "gemm_w4_tile_kernel", "moe_gate_up_kernel", "moe_down_kernel"):
        assert sum(part in name for name, _ in rings) >= 12, part


def test_nothing_is_spilled_and_no_fp32_is_packed(asm_files):
    checked = 0
    for path in asm_files:
        text = open(path).read()
        assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", text)
        for name, body in re.findall(r"\.name:\s+(_Z\S+)\n(.*?)\.wavefront_size", text, re.S):
            assert int(re.search(r"\.vgpr_spill_count:\s+(\d+)", body).group(1)) == 0, name
            checked += 1
    assert checked > 200

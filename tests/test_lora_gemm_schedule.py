"""Schedule invariants of the 192-row adapter GEMM (lora_gemm.hip::gemm_tall_lora_kernel), checked on the compiled gfx950
assembly (CPU only: hipcc cross-compiles).

The kernel waits for a stage with `s_waitcnt vmcnt(5)`: memory operations complete in issue order, so the wait is right only if
a group issues exactly its five loads and nothing else stands between them, spills among it; and the first half's products
must stand before the group's barrier, or the operands' reads are waited for with nothing to do."""
import os
import re
import shutil
import subprocess

import pytest

from flyai_amd import build as B

HIPCC = B.HIPCC if os.path.exists(B.HIPCC) else shutil.which("hipcc")
pytestmark = pytest.mark.skipif(HIPCC is None, reason="hipcc not available")
VMEM = re.compile(r"\s+(global_\w+|buffer_\w+|scratch_\w+|flat_\w+)")


@pytest.fixture(scope="module")
def bodies(tmp_path_factory):
    out = tmp_path_factory.mktemp("asm") / "lora_gemm.s"
    flags = [f for f in B.FLAGS if f != "-fPIC"]
    r = subprocess.run([HIPCC, *flags, "-S", "--cuda-device-only", "-x", "hip", os.path.join(B.CSRC, "lora_gemm.hip"), "-o", str(out)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    text = out.read_text()
    names = re.findall(r"\n(_ZN5flyai21gemm_tall_lora_kernel\w+):", text)
    assert len(names) == 2
    return [text[text.index("\n" + n + ":"):text.index(".Lfunc_end", text.index("\n" + n + ":"))].split("\n") for n in names]


def test_groups(bodies):
    for body in bodies:
        assert not any("scratch_" in line and line.startswith("\t") and "\t." not in line for line in body)
        waits = [i for i, line in enumerate(body) if re.match(r"\s+s_waitcnt vmcnt\(5\)", line)
                 and any("s_barrier" in near for near in body[i:i + 8])]
        assert len(waits) == 5                                    # three groups of the loop, two behind it
        for a, b in zip(waits, waits[1:3]):
            ops = [m[1] for m in map(VMEM.match, body[a:b]) if m]
            assert ops == ["global_load_lds_dwordx4"] * 5
            kinds = [m[1] for m in (re.match(r"\s+(s_barrier|v_mfma)", line) for line in body[a:b]) if m]
            assert kinds.count("s_barrier") == 1 and kinds[0] == "s_barrier" and kinds.count("v_mfma") == 24

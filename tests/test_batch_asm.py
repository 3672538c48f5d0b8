"""The key loops of attn_batch.hip count the copies in flight (s_waitcnt vmcnt(n)): any other vector memory access between
them would make the count wrong. The compiler's own would be spills, so the compiled kernels must have none. CPU only
(hipcc cross-compiles)."""
import os
import re
import shutil
import subprocess

import pytest

from moearc_amd import build

KERNELS = {f"moearc_attn_batch_{p}d{d}_k" for p in ("", "precise_") for d in (2, 4, 8)}


def scratch_bytes(assembly: str) -> dict:
    """Scratch bytes by kernel, as the assembly's comments state them."""
    out, kernel = {}, None
    for line in assembly.splitlines():
        m = re.match(r"(moearc_\w+):", line)
        if m:
            kernel = m.group(1)
        m = re.match(r"; ScratchSize: (\d+)", line)
        if m and kernel:
            out[kernel] = int(m.group(1))
    return out


def test_reads_the_compilers_figures():
    assert scratch_bytes("moearc_a_k:\n\ts_endpgm\n; ScratchSize: 0\nmoearc_b_k:\n; ScratchSize: 12\n") == {"moearc_a_k": 0, "moearc_b_k": 12}


@pytest.mark.skipif(not (shutil.which("hipcc") or os.path.exists(os.path.join(build.ROCM, "bin", "hipcc"))), reason="no hipcc")
def test_the_key_loops_kernels_spill_nothing(tmp_path):
    src, out = tmp_path / "kernels.hip", tmp_path / "kernels.s"
    src.write_text('#include "prefill.hip"\n#include "attn_batch.hip"\n')
    hipcc = shutil.which("hipcc") or os.path.join(build.ROCM, "bin", "hipcc")
    flags = [f for f in build.HIPCC_FLAGS if f not in ("--genco", "--no-gpu-bundle-output")]
    subprocess.run([hipcc, *flags, "--cuda-device-only", "-S", "-I", build.CSRC, str(src), "-o", str(out)], check=True, capture_output=True)
    found = scratch_bytes(out.read_text())
    assert KERNELS <= set(found)
    assert {k: found[k] for k in KERNELS} == dict.fromkeys(KERNELS, 0)

"""The prompt form of int4_linear shares one counter between its copies to LDS, which are assembly, and its
weight loads, which the compiler places: a wait for some of them by number would hold only as long as every
load stays one instruction in its place.  In the emitted code the step's barrier therefore follows a wait for
all of them, with no request in between."""
import re
import subprocess

import pytest

from helm_amd import build as hb


def steps_wait_for_all(asm):
    """{kernel: whether the wait ahead of its first barrier is for everything} of the prompt kernels."""
    found = {}
    for name, body in re.findall(r"^(\S*int4_gemm_kernel\S*):\s.*?$(.*?)^\.Lfunc_end", asm, re.S | re.M):
        ops = re.findall(r"^\s+([a-z]\w+)(.*)$", body, re.M)
        barrier = next(i for i, (op, _) in enumerate(ops) if op == "s_barrier")
        last = max(i for i in range(barrier) if ops[i][0] == "s_waitcnt" and "vmcnt" in ops[i][1])
        requests = [op for op, _ in ops[last:barrier] if op.startswith(("global_", "buffer_", "scratch_", "flat_"))]
        found[name] = "vmcnt(0)" in ops[last][1] and not requests
    return found


def test_a_step_of_a_prompt_waits_for_every_request(tmp_path):
    try:
        hipcc = hb._hipcc()
    except RuntimeError:
        pytest.skip("no hipcc")
    out = tmp_path / "int4.s"
    subprocess.run([hipcc, *hb.HIP_FLAGS, "--cuda-device-only", "-S", str(hb.CSRC / "int4.hip"), "-o", str(out)],
                   check=True, capture_output=True)
    found = steps_wait_for_all(out.read_text())
    assert len(found) == 24 and all(found.values()), found

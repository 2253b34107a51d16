"""Build-time invariant of the token mixers (CPU: hipcc cross-compiles gfx950 and reports per-kernel resources): no kernel keeps
registers in scratch memory.  A reload from scratch waits on the counter that the next tile's loads from memory are still
pending on, so a handful of spilled registers in such a loop drains its prefetch (28 of them: 87 -> 132 us in wattn_dq_kernel)."""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "speech-separation_amd", "csrc")


@pytest.mark.parametrize("src,kernels", [("wattn", 65), ("recur", 28), ("rotary", 14)])
def test_no_kernel_needs_scratch(src, kernels, tmp_path):
    if shutil.which("hipcc") is None:
        pytest.skip("hipcc not on PATH")
    # the command that make runs for this file, on the device side alone
    r = subprocess.run(["make", "-n", "-W", src + ".hip", src + ".o"], cwd=CSRC, capture_output=True, text=True)
    line = next(x for x in r.stdout.replace("\\\n", " ").splitlines() if src + ".hip" in x)
    cmd = [x for x in line.split() if x != "-c" and not x.endswith(".o") and x != "-o"]
    r = subprocess.run(cmd + ["--cuda-device-only", "-Rpass-analysis=kernel-resource-usage", "-c", "-o", str(tmp_path / "x")],
                       cwd=CSRC, capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stderr[-2000:]
    names = re.findall(r"remark: .*Function Name: (\S+)", r.stderr)
    scratch = re.findall(r"remark: .*ScratchSize \[bytes/lane\]: (\d+)", r.stderr)
    spilled = re.findall(r"remark: .*VGPRs Spill: (\d+)", r.stderr)
    assert len(names) == len(scratch) == len(spilled) >= kernels, (len(names), len(scratch))
    assert not {n: (s, v) for n, s, v in zip(names, scratch, spilled) if s != "0" or v != "0"}

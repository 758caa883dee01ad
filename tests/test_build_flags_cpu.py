"""Every HIP source is compiled without packed float32 instructions, some of whose forms have given wrong results on gfx950."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "marl_amd", "csrc")


def test_no_hip_source_is_compiled_with_packed_float32_instructions():
    lines = subprocess.run(["make", "-n", "-B", "-C", CSRC], capture_output=True, text=True, check=True).stdout.splitlines()
    compiled = [line for line in lines if " -c " in line and ".hip" in line]
    sources = sorted(f for f in os.listdir(CSRC) if f.endswith(".hip"))
    assert sorted(s for line in compiled for s in sources if f" {s} " in line) == sources
    for line in compiled:
        assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in line, line

"""Every HIP source is compiled without the packed fp32 instructions, whatever CXXFLAGS a caller brings."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cradle_vae_amd", "csrc")
FLAG = "-Xclang -target-feature -Xclang -packed-fp32-ops"


def _compile_lines(*args):
    out = subprocess.run(["make", "-n", "-B", "-C", CSRC, *args], check=True, capture_output=True, text=True).stdout
    return [line for line in out.splitlines() if " -c " in line and ".hip" in line]


def test_scalar_fp32_in_every_source():
    sources = [f for f in os.listdir(CSRC) if f.endswith(".hip")]
    for extra in ((), ("CXXFLAGS=-O2 -std=c++17 -fPIC --offload-arch=gfx950",)):
        lines = _compile_lines(*extra)
        assert len(lines) == len(sources) and len(sources) > 10
        for line in lines:
            assert FLAG in line, line
    for f in os.listdir(CSRC):
        if f.endswith((".hip", ".h")):
            text = open(os.path.join(CSRC, f)).read()
            assert not any("v_pk_%s_f32 " % op in text for op in ("add", "mul", "fma")), f

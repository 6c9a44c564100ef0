"""Every HIP compilation of the library is made without packed fp32 arithmetic: hipcc -O3 forms v_pk_add / mul / fma_f32 out of ordinary float
code by itself, and some of their forms have given wrong results on MI355X.  (Reads the build's own command lines; nothing is compiled.)"""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FLAG = "-Xclang -target-feature -Xclang -packed-fp32-ops"


@pytest.mark.parametrize("kdefs", ["", "-DRAYHS_DEV_KNOBS"])
def test_every_device_compilation_switches_packed_fp32_off(kdefs):
    out = subprocess.run(["make", "-C", os.path.join(ROOT, "rayhs_amd", "csrc"), "-n", "-B", f"KDEFS={kdefs}"], capture_output=True, text=True, check=True).stdout
    device = [l for l in out.split("\n") if "--offload-arch=" in l and " -c " in l]
    assert sum("trace_kernel.hip" in l for l in device) == 2 and any("abi.cpp" in l for l in device), out    # both variants of the kernels, and the launches
    for line in device:
        assert FLAG in line, line


def test_objects_are_rebuilt_when_the_build_file_changes():
    # a flag that changes has to reach the library: objects older than the build file are compiled again
    csrc = os.path.join(ROOT, "rayhs_amd", "csrc")
    out = subprocess.run(["make", "-C", csrc, "-n", "-W", "Makefile"], capture_output=True, text=True, check=True).stdout
    for name in ("trace_fast.o", "trace_exact.o", "abi.o", "host_scene.o", "bvh_build.o"):
        assert any(f"/{name}" in l and " -c " in l for l in out.split("\n")), name


def test_the_assembly_rewriting_build_compiles_its_kernels_the_same_way():
    text = open(os.path.join(ROOT, "tools", "build_asm_rewrite.sh")).read()
    assert FLAG in next(l for l in text.split("\n") if "--offload-arch=" in l)

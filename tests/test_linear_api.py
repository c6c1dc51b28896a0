"""The C entries of linear attention and the 4-bit projections on the CPU: compiled as host code, the HIP runtime and the launches
replaced by ones that write down what is called (linear_api.cpp)."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "..", "bitgpu_amd", "csrc")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="no hipcc")
def test_entries_against_a_stand_in_for_the_runtime(tmp_path):
    objects = []
    for src in (os.path.join(CSRC, "linear_api.hip"), os.path.join(HERE, "linear_api.cpp")):
        objects.append(str(tmp_path / (os.path.basename(src) + ".o")))
        subprocess.run([HIPCC, "-x", "hip", "--offload-arch=gfx950", "--offload-host-only", "-std=c++17", "-O1", "-g", "-fPIC", "-Wno-unused-result",
                        "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-c", src, "-o", objects[-1]], check=True)
    exe = str(tmp_path / "linear_api")
    subprocess.run(["g++", *objects, "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr

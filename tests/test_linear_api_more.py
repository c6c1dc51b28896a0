"""The C entries of linear attention on the CPU, continued (linear_api_more.cpp; compiled as test_linear_api.py does)."""
import os
import subprocess

import pytest

from tests.test_linear_api import CSRC, HERE, HIPCC


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="no hipcc")
def test_entries_against_a_stand_in_for_the_runtime(tmp_path):
    objects = []
    for src in (os.path.join(CSRC, "linear_api.hip"), os.path.join(HERE, "linear_api_more.cpp")):
        objects.append(str(tmp_path / (os.path.basename(src) + ".o")))
        subprocess.run([HIPCC, "-x", "hip", "--offload-arch=gfx950", "--offload-host-only", "-std=c++17", "-O1", "-g", "-fPIC",
                        "-Wno-unused-result", "-Wno-unused-function", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                        "-c", src, "-o", objects[-1]], check=True)
    exe = str(tmp_path / "linear_api_more")
    subprocess.run(["g++", *objects, "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr

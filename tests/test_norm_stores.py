"""Which rows of the norm behind a fold leave by buffer stores, which need 4-byte boundaries (no GPU).

tests/cpp/norm_stores.cpp compiles the planning as it is (vrank_fused.cpp) and goes through widths, strides and types: where
the streaming kernels are chosen, every piece of every stored row begins on a 4-byte boundary."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "megray_amd", "csrc")
SOURCES = ["vrank_fused.cpp", "megray_core.cpp", "bootstrap_client.cpp", "bootstrap_server.cpp"]


def test_streamed_rows_store_on_four_byte_boundaries(tmp_path):
    gxx = shutil.which("g++")
    rocm_include = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "include")
    if not gxx or not os.path.exists(os.path.join(rocm_include, "hip", "hip_runtime_api.h")):
        pytest.skip("needs g++ and the HIP runtime API headers")
    exe = str(tmp_path / "norm_stores")
    cmd = [gxx, "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=undefined", "-pthread",
           "-D__HIP_PLATFORM_AMD__=1", f"-I{ROOT}/include", f"-I{CSRC}", f"-I{rocm_include}",
           os.path.join(ROOT, "tests", "cpp", "norm_stores.cpp")]
    build = subprocess.run(cmd + [os.path.join(CSRC, s) for s in SOURCES] + ["-o", exe], capture_output=True, text=True, timeout=300)
    assert build.returncode == 0, build.stderr[-4000:]
    run = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.startswith("ok "), run.stdout[-2000:] + run.stderr[-2000:]

"""Calls on sequences that have evicted tokens, on the CPU:
tests/host/evicted_check.cpp includes the library's source and answers its launches
and graphs."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")


@pytest.mark.skipif(shutil.which("g++") is None or not os.path.isdir(os.path.join(ROCM, "include", "hip")),
                    reason="needs g++ and the HIP headers")
def test_sequences_that_have_evicted_tokens(tmp_path):
    exe = tmp_path / "evicted_check"
    csrc = os.path.join(HERE, "..", "qwen3.8_27b_in_rust_amd", "csrc")
    build = subprocess.run(["g++", "-O1", "-g", "-std=c++17", "-D__HIP_PLATFORM_AMD__=1", f"-I{ROCM}/include", f"-I{csrc}",
                            "-o", str(exe), os.path.join(HERE, "host", "evicted_check.cpp"),
                            os.path.join(csrc, "host", "q38_gguf.cpp"),
                            f"-L{ROCM}/lib", "-lamdhip64", f"-Wl,-rpath,{ROCM}/lib", "-ldl"],
                           capture_output=True, text=True)
    assert build.returncode == 0, build.stderr[-2000:]
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stdout[-2000:]
    assert "evicted ok" in run.stdout

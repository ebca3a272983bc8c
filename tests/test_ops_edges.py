"""The dense operators at their edges, as far as no GPU is needed."""
import os
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


def test_wait_limit_refuses(built_lib):
    assert built_lib.fv_ops_wait_limit(-2) == 1 and b"cycles" in built_lib.fv_last_error()
    assert built_lib.fv_ops_wait_limit(-1) == 0


def test_threads_that_ask_for_different_shared_memory(tmp_path):
    """Whichever thread sets a kernel's limit last, every size that was ever allowed stays allowed."""
    exe = tmp_path / "smem_limit_threads"
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    subprocess.run(["g++", "-std=c++17", "-pthread", f"-I{cuda}/include", f"-I{ROOT}/flyvec_b200/csrc", str(ROOT / "tests" / "smem_limit_threads.cpp"),
                    "-o", str(exe)], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stdout

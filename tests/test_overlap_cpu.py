"""Whether strided operands share memory: the host's check, under AddressSanitizer + UBSan (CPU only)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_shared_bytes_of_strided_blocks(tmp_path):
    exe = tmp_path / "overlap_checks"
    build = subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                            "-static-libasan", "-static-libubsan", "-I", os.path.join(ROOT, "csrc"),
                            os.path.join(ROOT, "tests", "native", "overlap_checks.cpp"), "-o", str(exe)],
                           capture_output=True, text=True)
    assert build.returncode == 0, build.stderr[-4000:]
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "overlap checks passed" in run.stdout, (run.stdout + run.stderr)[-4000:]
    print(run.stdout)

"""The streaming kernels' ring of copies when a wait runs out (no GPU: the protocol's own
code against a model of its barriers)."""

import os
import subprocess

from conftest import REPO


def test_no_copy_is_left_in_flight_when_a_wait_runs_out(tmp_path):
    exe = str(tmp_path / "ring_host_check")
    subprocess.run(["nvcc", "-std=c++17", "-O2", "-I", os.path.join(REPO, "blockstreamer_b200", "csrc"),
                    os.path.join(REPO, "tests", "native", "ring_host_check.cu"), "-o", exe], check=True)
    res = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert res.stdout.strip() == "BAD 0" and res.returncode == 0, res.stdout

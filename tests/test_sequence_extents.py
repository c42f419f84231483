"""What the host layer's operators of networks over sequences ask of their arrays' extents (no GPU): a C++ program
with entry points that only count their calls, built with the operators' own source."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HOST = os.path.join(ROOT, "minerva_amd", "host")


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("extents") / "sequence_extents_test")
    srcs = [os.path.join(ROOT, "tests", "host_cpu", "sequence_extents_test.cpp"), os.path.join(HOST, "hip_sequence_ops.cpp")]
    build = subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-I" + HOST, "-I" + os.path.join(ROOT, "include")] + srcs + ["-o", exe],
                           capture_output=True, text=True)
    assert build.returncode == 0, build.stderr[-3000:]
    return exe


@pytest.mark.parametrize("what", ["mixed", "empty"])
def test_extents(program, what):
    run = subprocess.run([program, what], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and run.stdout.strip() == "OK", (run.returncode, run.stdout + run.stderr)

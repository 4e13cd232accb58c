"""tfcc::rocm::generation of the C++ host layer (tests/cpp/generation_tests.cpp): refusals on the CPU, known answers on the GPU."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DRIVER = os.path.join(ROOT, "wechat-tfcc_amd", "host", "build", "generation_tests")


def run(mode):
    if not os.path.exists(DRIVER):
        subprocess.check_call(["make", "-s", "-C", os.path.join(ROOT, "wechat-tfcc_amd", "host"), "build/generation_tests"])
    res = subprocess.run([DRIVER, mode], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=100)
    assert res.returncode == 0 and "all passed" in res.stdout, res.stdout[-2000:]


def test_refusals():
    run("cpu")


@pytest.mark.gpu
def test_known_answers():
    run("gpu")

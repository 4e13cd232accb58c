"""Norms, 4-bit caches, copies and shaped scores of the C++ host layer (tests/cpp/serving_tests.cpp): refusals on the CPU, known answers on the GPU; and how
attention over 4-bit caches is dealt out (tests/cpp/serving_plan_tests.cpp), on the CPU."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HOST = os.path.join(ROOT, "wechat-tfcc_amd", "host")


def run(name, *mode):
    driver = os.path.join(HOST, "build", name)
    if not os.path.exists(driver):
        subprocess.check_call(["make", "-s", "-C", HOST, "build/" + name])
    res = subprocess.run([driver, *mode], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=100)
    assert res.returncode == 0 and "all passed" in res.stdout, res.stdout[-2000:]


def test_refusals():
    run("serving_tests", "cpu")


def test_plan():
    subprocess.check_call(["make", "-s", "-C", HOST, "build/serving_plan_tests"])
    run("serving_plan_tests")


@pytest.mark.gpu
def test_known_answers():
    run("serving_tests", "gpu")

"""The tanh of capped scores as the kernels form it (tests/cpp/score_tanh_tests.cpp), on the CPU."""
import os
import subprocess

HOST = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "wechat-tfcc_amd", "host")


def test_against_64_bits():
    subprocess.check_call(["make", "-s", "-C", HOST, "build/score_tanh_tests"])
    res = subprocess.run([os.path.join(HOST, "build", "score_tanh_tests")], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=100)
    assert res.returncode == 0 and "all passed" in res.stdout, res.stdout[-2000:]

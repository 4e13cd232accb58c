"""When attention over a paged cache takes the longest sequences first, and which launch joins its pieces (tests/cpp/attention_order_tests.cpp), on the CPU."""
import os
import subprocess

HOST = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "wechat-tfcc_amd", "host")


def test_both_sides_of_the_lines():
    subprocess.check_call(["make", "-s", "-C", HOST, "build/attention_order_tests"])
    res = subprocess.run([os.path.join(HOST, "build", "attention_order_tests")], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=100)
    assert res.returncode == 0 and "all passed" in res.stdout, res.stdout[-2000:]

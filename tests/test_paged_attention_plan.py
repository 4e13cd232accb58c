"""How attention over a paged cache is dealt out, on the CPU (tests/cpp/paged_attention_plan_tests.cpp)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_tiles_and_pieces_hold_every_row_and_key():
    host = os.path.join(ROOT, "wechat-tfcc_amd", "host")
    subprocess.check_call(["make", "-s", "-C", host, "build/paged_attention_plan_tests"])
    res = subprocess.run([os.path.join(host, "build", "paged_attention_plan_tests")], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert res.returncode == 0 and "all passed" in res.stdout, res.stdout[-2000:]

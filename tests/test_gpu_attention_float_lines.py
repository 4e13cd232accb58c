"""Plain attention over a float32 cache: calls of fewer than 18000 rows over fewer than 2048 keys run on the fp32 operations, which lose nothing of a row; and where the lines of
that rule lie (tests/cpp/float_cache_plan_tests.cpp), on the CPU."""
import os
import subprocess

import numpy as np
import pytest

from test_gpu_paged_attention import Made

HOST = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "wechat-tfcc_amd", "host")


def test_lines():
    subprocess.check_call(["make", "-s", "-C", HOST, "build/float_cache_plan_tests"])
    res = subprocess.run([os.path.join(HOST, "build", "float_cache_plan_tests")], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=100)
    assert res.returncode == 0 and "all passed" in res.stdout, res.stdout[-2000:]


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,chunks,heads,kv,size,page", [([1500, 1400], [256, 256], 32, 8, 128, 32), ([1024, 1024], [512, 512], 12, 12, 64, 16), ([1500], [700], 16, 16, 64, 20),
                                                               ([2000, 1999], [200, 148], 24, 4, 96, 16)])
def test_small_parts_of_a_row_are_kept(pkg, T, lengths, chunks, heads, kv, size, page):
    """Scores and results that come from parts of keys, queries and values 2^-34 below their row's largest."""
    mean = -(-sum(chunks) // len(chunks))
    assert 8192 <= mean * len(chunks) * heads < 18000
    m = Made(pkg, "f32", lengths, chunks, heads, kv, size, page, 7)
    small = np.float32(2.0 ** -34)
    m.cache[0][..., 1:] *= small
    m.q[..., 1:] /= small
    m.q[..., 0] = 0
    m.check(T)
    m.cache[1][..., 1:] *= small
    want = m.run(T)
    got, whole = T.n(want)[..., 1:], m.cache[1]
    # the first values are not there: the others are those of a cache without them
    m.cache[1] = whole.copy()
    m.cache[1][..., 0] = 0
    m.cache[1][..., 1:] /= small
    without = T.n(m.run(T))[..., 1:]
    assert np.array_equal(got, without * small)  # powers of two

"""Products of two MXFP4 matrices whose C is so large that it is stored past the caches, in each size of tile, exact: one scale everywhere, so every partial
sum is a multiple of a quarter below 2^24 quarters."""
import numpy as np
import pytest

import mx_support as mx
from test_gpu_mx_gemm import operand, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k", (96, 1024, 2560))
def test_results_past_the_caches_are_exact(gpu, k):
    m, n = 7105, 7099
    rng = np.random.default_rng(k)
    a, b = operand(rng, m, k, low=127, high=128), operand(rng, n, k, low=127, high=128)
    got = run(gpu, "device", a, b, k, 1.0, 0.0, np.full(m * n, np.nan, np.float32), m, n, n, 1).reshape(m, n)
    want = mx.values(a[0], a[1]).astype(np.float32) @ mx.values(b[0], b[1]).astype(np.float32).T
    assert np.array_equal(got, want)

"""Products of two MXFP4 matrices whose results lie below fp32's smallest normal number, in every kernel: numbers like any others, exact down to 2^-149."""
import numpy as np
import pytest

import mx_support as mx
from test_gpu_mx_gemm import run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,k", ((16, 96, 640), (70, 40, 640), (70, 40, 613), (300, 4096, 640), (1500, 1500, 1600), (2048, 4096, 2048), (3500, 4096, 2592)))
def test_results_below_the_smallest_normal_number(gpu, m, n, k):
    """Rows of A hold one to four ones, columns of B one value of 1 to 3 times 2^-126 to 2^-149 and less, that share that block."""
    blocks = -(-k // 32)
    rng = np.random.default_rng(k)
    a, b = np.zeros((m, k), np.uint8), np.full((n, k), 2, np.uint8)
    count = rng.integers(1, 5, size=m)
    block = rng.integers(0, k // 32, size=m)
    for i in range(m):
        a[i, 32 * block[i]:32 * block[i] + count[i]] = 2
    b[:] = rng.choice(np.array([2, 4, 5], np.uint8), size=(n, 1))  # 1, 2, 3 all along a column
    low, high = rng.integers(0, 12, size=(m, blocks)), rng.integers(0, 14, size=(n, blocks))  # 2^-127 .. 2^-116 and 2^-13 .. 1
    sa, sb = low.astype(np.uint8), (114 + high).astype(np.uint8)
    op = lambda code, scales: (code, scales, *mx.store(code, scales, k + k % 2, blocks), k + k % 2, blocks)  # noqa: E731
    got = run(gpu, "device", op(a, sa), op(b, sb), k, 1.0, 0.0, np.full(m * n, np.nan, np.float32), m, n, n, 1).reshape(m, n)
    value = np.array([0, 0, 1, 0, 2, 3])[b[:, 0]]
    exponent = (low[np.arange(m), block] - 127)[:, None] + (high[:, block].T - 13)
    want = np.ldexp((count[:, None] * value[None, :]).astype(np.float64), exponent)
    assert (want < 2.0 ** -126).mean() > 0.3 and want.min() >= 2.0 ** -149
    assert np.array_equal(got.astype(np.float64), want)

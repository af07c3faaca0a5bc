"""Products of two MXFP4 matrices where rows and columns end: K just past what is read without a copy, rows that begin on odd bytes, whole and partial blocks
at the end of rows of every length, and last columns of C that do not fill a vector, written and added to."""
import numpy as np
import pytest

from test_gpu_mx_gemm import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k", (2047, 2048, 2049, 2050, 2082, 2303, 2304, 2305, 4099))
@pytest.mark.parametrize("m,n", ((20, 300), (100, 300)))
def test_rows_on_odd_bytes(gpu, m, n, k):
    even = k + k % 2
    check(gpu, "device", np.random.default_rng(k), m, n, k, beta=0.25, lda=even + 2, lsa=-(-k // 32) + 3, ldb=even + 6, lsb=-(-k // 32) + 1)


@pytest.mark.parametrize("k", (1, 2, 31, 32, 33, 63, 64, 65, 95, 193, 223, 224, 225, 255, 256, 257, 287, 288, 289, 481, 500, 511, 513))
def test_every_kind_of_end(gpu, k):
    """Of rows shorter than a load of codes or scales, and of longer ones."""
    rng = np.random.default_rng(k)
    for m, n in ((3, 70), (70, 90)):
        check(gpu, "device", rng, m, n, k)
        check(gpu, "device", rng, m, n, k, lda=k + k % 2 + 2, ldb=k + k % 2 + 4)


@pytest.mark.parametrize("n", (2051, 2065, 2110, 2176))
@pytest.mark.parametrize("m,k", ((2176, 1024), (3300, 2600)))
def test_last_columns_of_large_tiles(gpu, m, n, k):
    rng = np.random.default_rng(n)
    n += 2000 if m > 3000 else 0
    check(gpu, "device", rng, m, n, k)
    check(gpu, "device", rng, m, n, k, alpha=-0.5, beta=2.0, rsc=n + 1)

"""Products and sums through an index into operands of nearly 3 GiB, as far as the streaming kernels' 32-bit offsets go, and of a row more, which the kernel for any layout takes. Rows are
picked from both ends; everything else is NaN. Sums of whole numbers: exact."""
import numpy as np
import pytest

import grouped_support as gs
import skl_amd
from skl_amd import DeviceBuffer
from test_gpu_grouped_tiles import put

pytestmark = pytest.mark.gpu

PITCH, K = 40000, 64
BELOW = (0xC0000000 // 2 - K - 1) // PITCH  # the most rows with (rows * PITCH + K) * 2 below 3 GiB


@pytest.fixture(scope="module")
def operand(gpu):
    """(buffer, rows that hold numbers, those numbers)."""
    rng = np.random.default_rng(3)
    buf = DeviceBuffer(2 * (BELOW + 2) * PITCH)
    gpu.skl_hip_memset(buf, 0xFF, buf.nbytes)
    at = np.array([0, 1, BELOW // 3, (1 << 31) // (2 * PITCH), (1 << 31) // (2 * PITCH) + 1, BELOW - 2, BELOW - 1])  # bytes below and beyond 2^31
    x = gs.bits(rng.integers(-4, 5, (len(at), K)), "bf16")
    for r, v in zip(at, x):
        put(gpu, buf.offset(2 * int(r) * PITCH), v)
    yield buf, at, gs.values(x, "bf16")
    buf.free()


def picked(rng, m, at, x, rows):
    """An index of m rows, some outside, and what it picks."""
    which = rng.integers(0, len(at), m)
    index, values = at[which], x[which]
    out = rng.random(m) < 0.2
    index[out], values[out] = rng.choice([-1, rows, rows + 1, -2 ** 31, 2 ** 31 - 1], out.sum()), 0.0
    return index.astype(np.int32), values


@pytest.mark.parametrize("rows", (BELOW, BELOW + 1), ids=("below", "beyond"))
@pytest.mark.parametrize("m,n", ((30, 72), (2600, 4096)))  # tiles of 64 and of 256 rows
def test_products(gpu, operand, m, n, rows):
    buf, at, x = operand
    rng = np.random.default_rng(m)
    index, picks = picked(rng, m, at, x, rows)
    w = gs.bits(rng.integers(-4, 5, (2, n, K)), "bf16")
    offsets = np.array([0, m // 3, m - 1], np.int32)
    di, dw, do, c = DeviceBuffer.from_array(index), DeviceBuffer.from_array(w), DeviceBuffer.from_array(offsets), DeviceBuffer(4 * m * n)
    for strides in ((1, K), (n, 1)):
        gpu.skl_hip_memset(c, 0, c.nbytes)
        wv = gs.values(w, "bf16") if strides[0] == 1 else gs.values(w, "bf16").reshape(2, K, n).transpose(0, 2, 1)
        gpu.skl_gemm_grouped_bf16_bf16rc_f32_gfx950(2, do, m, n, K, 1.0, buf, PITCH, di, rows, dw, *strides, n * K, 0.0, c, n)
        assert gpu.skl_hip_synchronize() == 0
        skl_amd.check_error()
        want = np.concatenate([picks[:m // 3] @ wv[0].T, picks[m // 3:m - 1] @ wv[1].T, np.zeros((1, n))])
        assert np.array_equal(c.download(np.float32).reshape(m, n), want), strides


@pytest.mark.parametrize("rows", (BELOW, BELOW + 1), ids=("below", "beyond"))
@pytest.mark.parametrize("total,n", ((100, 72), (900, 9000)))  # tiles of 128 x 128 and of 256 x 256
def test_sums(gpu, operand, total, n, rows):
    buf, at, x = operand
    rng = np.random.default_rng(total)
    index, picks = picked(rng, total, at, x, rows)
    y = gs.bits(rng.integers(-4, 5, (total, n)), "bf16")
    yv = gs.values(y, "bf16")
    offsets = np.array([0, total // 3, total // 3, total - 1, total - 1], np.int32)
    di, dy, do, c = DeviceBuffer.from_array(index), DeviceBuffer.from_array(y), DeviceBuffer.from_array(offsets), DeviceBuffer(4 * 4 * K * n)
    big, small = (buf, PITCH, di, rows), (dy, n, None, 0)
    for turned in (False, True):
        m_, n_ = (n, K) if turned else (K, n)
        a, b = (small, big) if turned else (big, small)
        gpu.skl_gemm_groupedk_bf16c_bf16_f32_gfx950(4, do, m_, n_, total, 1.0, *a, *b, 0.0, c, n_, m_ * n_)
        assert gpu.skl_hip_synchronize() == 0
        skl_amd.check_error()
        got = c.download(np.float32).reshape(4, m_, n_)
        for e in range(4):
            sums = picks[offsets[e]:offsets[e + 1]].T @ yv[offsets[e]:offsets[e + 1]]
            assert np.array_equal(got[e], sums.T if turned else sums), (e, turned)

"""MXFP4 conversions whose rows and blocks are more than a launch has threads for: beyond 2^32 a launch is refused, or runs what is left of the number in 32 bits. The source's values lie on one another (a distance of zero), so that only what is
written is large; looked at where one launch's part ends and the next begins, and at the ends."""
import numpy as np
import pytest

import mx_support as mx
import skl_amd
from skl_amd import DeviceBuffer

pytestmark = pytest.mark.gpu


def some(lib, buf, at, count):
    out = np.empty(count, np.uint8)
    assert lib.skl_hip_memcpy_d2h(out.ctypes.data, buf.offset(at), count) == 0
    return out


def check(lib, m, k, rs, cs, places):
    """Row i of the source is its element i * rs, k times over. `places`: (row, value), multiples of 32."""
    values = mx.to_bf16(np.random.default_rng(m).normal(size=(m - 1) * rs + 1).astype(np.float32))
    rows, blocks = k // 2, k // 32
    src, dst, scales = DeviceBuffer.from_array(values), DeviceBuffer(m * rows), DeviceBuffer(m * blocks)
    try:
        lib.skl_cvt_bf16rc_mxf4e2m1_gfx950(m, k, src, rs, cs, dst, k, scales, blocks)
        lib.skl_hip_synchronize()
        skl_amd.check_error()
        for i, p in places:
            code, scale = mx.quantise(np.full((1, 32), mx.of_bf16(values[i * rs:i * rs + 1])[0], np.float64))
            assert np.array_equal(some(lib, dst, i * rows + p // 2, 16), np.full(16, code[0, 0] * 17, np.uint8)), (i, p)
            assert some(lib, scales, i * blocks + p // 32, 1)[0] == scale[0, 0], (i, p)
        back = DeviceBuffer(2 * m)  # each row on one value, all of them alike
        lib.skl_cvt_mxf4e2m1_bf16rc_gfx950(m, k, dst, k, scales, blocks, back, 1, 0)
        lib.skl_hip_synchronize()
        skl_amd.check_error()
        got = mx.of_bf16(back.download(np.uint16, m))
        for i, _ in places:
            code, scale = mx.quantise(np.full((1, 32), mx.of_bf16(values[i * rs:i * rs + 1])[0], np.float64))
            assert got[i] == mx.values(code, scale)[0, 0]
        back.free()
    finally:
        for b in (src, dst, scales):
            b.free()


def test_as_many_blocks_as_fill_two_launches(gpu):
    """2^30 blocks in 2^15 rows."""
    m, k = 1 << 15, 1 << 20
    check(gpu, m, k, 3, 0, [(0, 0), (0, k - 32), (m // 2 - 1, k - 32), (m // 2, 0), (m // 2, k // 2), (m - 1, 0), (m - 1, k - 32)])


def test_a_row_longer_than_a_launch(gpu):
    k = (1 << 34) + 4096
    check(gpu, 1, k, 1, 0, [(0, 0), (0, 1 << 33), (0, (1 << 34) - 32), (0, 1 << 34), (0, k - 32)])


def test_columns_longer_than_a_launch(gpu):
    k = (1 << 31) + 608
    check(gpu, 3, k, 1, 0, [(i, p) for i in range(3) for p in (0, 1 << 29, (1 << 30) - 32, 1 << 30, (1 << 31) - 32, 1 << 31, k - 32)])

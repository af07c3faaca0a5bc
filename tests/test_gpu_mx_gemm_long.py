"""Products of two MXFP4 matrices with more rows or columns than a launch has threads for, looked at where one launch's part ends and the next begins, around what is left
of a number of threads in 32 bits, and at the ends."""
import numpy as np
import pytest

import skl_amd
from skl_amd import DeviceBuffer

pytestmark = pytest.mark.gpu


def check(lib, rows, k, other, places):
    """`rows` rows of ones in one operand - twos at `places` - against one row of threes in the other; `other`: 'a' or 'b', the operand of one row."""
    codes, scales, c = DeviceBuffer(rows * k // 2), DeviceBuffer(rows * k // 32), DeviceBuffer(4 * rows)
    one, one_scales = DeviceBuffer.from_array(np.full(k // 2, 0x55, np.uint8)), DeviceBuffer.from_array(np.full(k // 32, 127, np.uint8))
    try:
        assert lib.skl_hip_memset(codes.ptr, 0x22, codes.nbytes) == 0 and lib.skl_hip_memset(scales.ptr, 127, scales.nbytes) == 0
        assert lib.skl_hip_memset(c.ptr, 0xFF, c.nbytes) == 0
        two = np.full(k // 2, 0x44, np.uint8)
        for at in places:
            assert lib.skl_hip_memcpy_h2d(codes.offset(at * (k // 2)), two.ctypes.data, two.size) == 0
        many, single = (codes, k, scales, k // 32), (one, k, one_scales, k // 32)
        a, b = (single, many) if other == "a" else (many, single)
        m, n = (1, rows) if other == "a" else (rows, 1)
        lib.skl_gemm_mxf4e2m1r_mxf4e2m1c_f32rc_gfx950(m, n, k, 1.0, *a, *b, 0.0, c, n, 1)
        lib.skl_hip_synchronize()
        skl_amd.check_error()
        piece = 1 << 26
        for first in range(0, rows, piece):
            got = np.empty(min(piece, rows - first), np.float32)
            assert lib.skl_hip_memcpy_d2h(got.ctypes.data, c.offset(4 * first), got.nbytes) == 0
            wrong = np.flatnonzero(got != 3.0 * k) + first
            assert wrong.tolist() == [at for at in sorted(places) if first <= at < first + piece], first
            assert (got[wrong - first] == 6.0 * k).all()
    finally:
        for buf in (codes, scales, c, one, one_scales):
            buf.free()


def test_more_rows_than_a_launch_has_tiles(gpu):
    rows = (1 << 30) + 197
    check(gpu, rows, 32, "b", [0, 63, 64, (1 << 28) - 1, 1 << 28, 1 << 29, (1 << 30) - 1, 1 << 30, (1 << 30) + 64, rows - 1])


def test_columns_in_two_slabs_and_more(gpu):
    rows = (1 << 29) + 333
    check(gpu, rows, 256, "a", [0, 63, 64, (1 << 28) - 1, 1 << 28, (1 << 29) - 1, 1 << 29, rows - 1])

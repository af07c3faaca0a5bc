"""Host threads that make the calls of two launches at once - the order of many picks, sums in parts - on one stream, whose scratch memory they share, and on a stream each."""
import ctypes as ct
import threading

import numpy as np
import pytest

import grouped_support as gs
import skl_amd
from skl_amd import DeviceBuffer

pytestmark = pytest.mark.gpu

PICKS, GROUPS, ROWS, COLS = 40000, 70, 5000, 128


class Work:
    def __init__(self, seed):
        rng = np.random.default_rng(seed)
        ids = rng.integers(-1, GROUPS, PICKS).astype(np.int32)
        self.want = gs.group_rows(ids, 2, GROUPS)
        a, b = (gs.bits(rng.integers(-4, 5, (ROWS, COLS)), "bf16") for _ in range(2))
        self.sums = gs.values(a, "bf16").T @ gs.values(b, "bf16")
        at = DeviceBuffer.from_array
        self.ids, self.a, self.b = at(ids), at(a), at(b)
        self.offsets, self.order, self.rows, self.place = (DeviceBuffer(4 * v) for v in (GROUPS + 1, PICKS, PICKS, PICKS))
        self.c = DeviceBuffer(4 * COLS * COLS)

    def enqueue(self, lib):
        lib.skl_group_rows_gfx950(PICKS, self.ids, 2, GROUPS, self.offsets, self.order, self.rows, self.place)
        lib.skl_gemm_groupedk_bf16c_bf16_f32_gfx950(1, None, COLS, COLS, ROWS, 1.0, self.a, COLS, None, 0, self.b, COLS, None, 0, 0.0, self.c, COLS, COLS * COLS)

    def check(self):
        offsets, order, rows, place = self.want
        assert np.array_equal(self.offsets.download(np.int32), offsets) and np.array_equal(self.place.download(np.int32), place)
        assert np.array_equal(self.order.download(np.int32)[:len(order)], order) and np.array_equal(self.rows.download(np.int32)[:len(rows)], rows)
        assert np.array_equal(self.c.download(np.float32).reshape(COLS, COLS), self.sums)


@pytest.mark.parametrize("together", (True, False), ids=("one stream", "a stream each"))
def test_two_threads(gpu, together):
    hip = ct.CDLL("libamdhip64.so.7")
    hip.hipStreamCreate.restype = hip.hipStreamDestroy.restype = ct.c_int
    work, streams, failed = [Work(1), Work(2)], [ct.c_void_p(), ct.c_void_p()], []
    assert gpu.skl_hip_synchronize() == 0  # the uploads
    for stream in streams:
        assert hip.hipStreamCreate(ct.byref(stream)) == 0
    start = threading.Barrier(2)

    def run(i):
        try:
            assert gpu.skl_hip_init(0) == 0
            gpu.skl_hip_set_pointer_mode(1)
            gpu.skl_hip_set_stream(streams[0 if together else i].value)
            start.wait(60)
            for _ in range(8):
                for _ in range(10):
                    work[i].enqueue(gpu)
                assert gpu.skl_hip_synchronize() == 0
                skl_amd.check_error()
                work[i].check()
        except BaseException as e:  # noqa: B902
            failed.append(e)
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for stream in streams:
        gpu.skl_hip_release_stream(stream.value)
        hip.hipStreamDestroy(stream)
    if failed:
        raise failed[0]

"""The order of picks by their groups (skl_group_rows) against its definition: every number is exact."""
import numpy as np
import pytest

import grouped_support as gs
import skl_amd
from skl_amd import DeviceBuffer

pytestmark = pytest.mark.gpu

FILL = -77


def call(lib, ids, per_row, groups, wanted=(True, True, True), mode="device"):
    """(offsets, order, rows, place) behind the call, None for what was not asked for."""
    ids = np.asarray(ids, np.int32)
    out = [np.full(groups + 1, FILL, np.int32)] + [np.full(max(len(ids), 1), FILL, np.int32) if w else None for w in wanted]
    if mode == "host":
        lib.skl_group_rows_gfx950(len(ids), ids, per_row, groups, *out)
        skl_amd.check_error()
        return out
    d_ids, bufs = DeviceBuffer.from_array(ids), [None if o is None else DeviceBuffer.from_array(o) for o in out]
    lib.skl_group_rows_gfx950(len(ids), d_ids, per_row, groups, *bufs)
    assert lib.skl_hip_synchronize() == 0
    skl_amd.check_error()
    return [None if b is None else b.download(np.int32, len(o)) for b, o in zip(bufs, out)]


def check(got, ids, per_row, groups):
    offsets, order, rows, place = gs.group_rows(ids, per_row, groups)
    assert np.array_equal(got[0], offsets)
    inside = len(order)
    for have, want in ((got[1], order), (got[2], rows)):
        if have is not None:
            assert np.array_equal(have[:inside], want)
            assert np.all(have[inside:] == FILL), "places behind the last group were written"
    if got[3] is not None and len(ids):
        assert np.array_equal(got[3][:len(ids)], place)


@pytest.mark.parametrize("mode", ("host", "device"))
@pytest.mark.parametrize("count,per_row,groups", [(0, 1, 5), (1, 1, 1), (1, 8, 4096), (7, 3, 2), (64, 8, 8), (128, 8, 128), (1023, 4, 65), (1024, 1, 64), (1025, 2, 63), (4096, 8, 257),
                                                  (4097, 6, 256), (10001, 8, 1000), (65536, 8, 256), (99999, 5, 4096)])
def test_against_the_definition(gpu, mode, count, per_row, groups):
    rng = np.random.default_rng(count + groups)
    ids = rng.integers(0, groups, count)
    ids[rng.random(count) < 0.1] = rng.choice([-1, groups, -2 ** 31, 2 ** 31 - 1])
    check(call(gpu, ids, per_row, groups, mode=mode), ids, per_row, groups)


@pytest.mark.parametrize("count,groups", [(2047, 40), (2048, 40), (2049, 40), (2049, 4096), (3000, 1), (300000, 3), (300000, 300), (700001, 2048)])
def test_one_workgroup_and_more(gpu, count, groups):
    ids = np.random.default_rng(count).integers(-1, groups, count)
    check(call(gpu, ids, 1, groups), ids, 1, groups)


@pytest.mark.parametrize("count", (5, 3000, 40000))
def test_one_group_takes_all_or_nothing(gpu, count):
    for ids, groups in ((np.zeros(count), 1), (np.full(count, 6), 7), (np.full(count, -1), 7), (np.arange(count) % 2 * 63, 64)):
        check(call(gpu, ids, 2, groups), ids, 2, groups)


@pytest.mark.parametrize("count", (33, 20000))
def test_outputs_that_are_not_wanted(gpu, count):
    rng = np.random.default_rng(count)
    ids = rng.integers(-1, 12, count)
    for wanted in ((False, False, False), (True, False, False), (False, True, False), (False, False, True)):
        check(call(gpu, ids, 4, 11, wanted), ids, 4, 11)


def test_a_large_count(gpu):
    rng = np.random.default_rng(3)
    ids = rng.integers(0, 300, 3_000_000)
    got = call(gpu, ids, 8, 300)
    order = np.argsort(ids, kind="stable")
    place = np.empty_like(order)
    place[order] = np.arange(len(order))
    assert np.array_equal(got[0], np.concatenate(([0], np.cumsum(np.bincount(ids, minlength=300)))))
    assert np.array_equal(got[1], order) and np.array_equal(got[2], order // 8) and np.array_equal(got[3], place)

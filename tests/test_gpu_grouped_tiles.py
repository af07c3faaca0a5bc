"""Products grouped by expert where their kernels change: every tile size, groups that end on and beside the ends of tiles, short and uneven sums, rows through an index, memory beyond 32 bits
of offsets. The comparisons are test_gpu_gemm_grouped's."""
import numpy as np
import pytest

import grouped_support as gs
import skl_amd
from skl_amd import DeviceBuffer
from test_gpu_gemm_grouped import run_grouped, run_groupedk

pytestmark = pytest.mark.gpu


def offsets_of(sizes, front=0):
    return (front + np.concatenate(([0], np.cumsum(sizes)))).astype(np.int32)


# (sizes of the groups, n): what skl_gemm_grouped takes in tiles of 256, 128 and 64 rows
LARGE = ([256, 257, 0, 65, 64, 700, 1, 128, 129, 512, 300, 63], 5000)
MIDDLE = ([128, 129, 0, 64, 65, 1, 127, 30, 100, 190], 4300)
SMALL = ([64, 65, 1, 0, 0, 63, 2, 128, 16, 40], 200)


@pytest.mark.parametrize("layout", ("col", "row"))
@pytest.mark.parametrize("sizes,n", (LARGE, MIDDLE, SMALL), ids=("256", "128", "64"))
@pytest.mark.parametrize("kind", ("bf16", "f16"))
def test_ends_of_tiles(gpu, kind, sizes, n, layout):
    for k, out in ((8, "f32"), (24, kind), (64, "f32"), (136, kind), (264, "f32")):
        for cols in (n, n - 3, max(8, n // 8 * 8 - 248)):
            if k > 64 and cols != n - 3:
                continue
            m = sum(sizes) + 9
            run_grouped(gpu, kind, out, m, cols, k, offsets_of(sizes, 4), len(sizes), layout=layout, seed=k + cols, pads=(0, -cols % 8 if layout == "row" else 0, 0))


@pytest.mark.parametrize("layout", ("col", "row"))
@pytest.mark.parametrize("sizes,n", (LARGE, MIDDLE, SMALL), ids=("256", "128", "64"))
def test_ends_of_tiles_with_an_index(gpu, sizes, n, layout):
    rng = np.random.default_rng(1)
    m = sum(sizes) + 5
    index = rng.integers(0, 333, m)
    index[rng.random(m) < 0.05] = -1
    run_grouped(gpu, "bf16", "f32", m, n // 8 * 8, 72, offsets_of(sizes), len(sizes), index=index, a_rows=333, layout=layout, seed=2)
    run_grouped(gpu, "bf16", "bf16", m, n // 8 * 8, 72, offsets_of(sizes), len(sizes), index=index, a_rows=333, layout=layout, alpha=0.5, beta=-1.0, pads=(8, 8, 8), seed=3)


@pytest.mark.parametrize("groups", (63, 64, 65, 200, 4096))
def test_many_groups(gpu, groups):
    rng = np.random.default_rng(groups)
    sizes = rng.integers(0, 5, groups)
    sizes[rng.integers(0, groups)] = 150
    for k in (40, 33):
        run_grouped(gpu, "bf16", "f32", int(sizes.sum()), 72, k, offsets_of(sizes), groups, seed=groups)
    if groups < 4096:
        run_groupedk(gpu, "bf16", "f32", 40, 72, int(sizes.sum()) + 3, offsets_of(sizes, 2), groups, seed=groups)
        run_groupedk(gpu, "bf16", "f32", 40, 71, int(sizes.sum()) + 3, offsets_of(sizes, 2), groups, seed=groups)


@pytest.mark.parametrize("groups,n,layout", ((64, 5118, "col"), (130, 2560, "row")))
def test_many_tiles_of_uneven_groups(gpu, groups, n, layout):
    """Many tiles of 256 rows, last lines of every length."""
    rng = np.random.default_rng(groups)
    share = rng.exponential(size=groups) ** 2 * (rng.random(groups) > 0.1)
    sizes = np.floor(share / share.sum() * 113 * groups).astype(int)
    sizes[groups // 2] += 113 * groups - sizes.sum()
    run_grouped(gpu, "bf16", "bf16", int(sizes.sum()) + 3, n, 16, offsets_of(sizes, 3), groups, layout=layout, seed=groups)
    # all in one group, the last: one lane holds all tiles
    sizes[:], sizes[-1] = 0, 113 * groups
    run_grouped(gpu, "bf16", "bf16", int(sizes.sum()), n, 8, offsets_of(sizes), groups, layout=layout, seed=groups)


LENGTHS = [0, 1, 31, 32, 33, 64, 65, 127, 128, 129, 0, 160, 300, 7]


@pytest.mark.parametrize("indexed", ((False, False), (False, True), (True, False), (True, True)), ids=str)
@pytest.mark.parametrize("kind", ("bf16", "f16"))
def test_sums_of_every_length(gpu, kind, indexed):
    """Tiles of 256 x 256 values of C, more than one of them, with ends in both directions."""
    total = sum(LENGTHS) + 6
    rng = np.random.default_rng(total)
    index = [rng.integers(-1, 90, total) if i else None for i in indexed]
    for m, n, out in ((264, 520, "f32"), (256, 256, kind), (72, 300, "f32")):
        pads = (-m % 8, -n % 8, 0)
        run_groupedk(gpu, kind, out, m, n, total, offsets_of(LENGTHS, 3), len(LENGTHS), index[0], 90 if indexed[0] else 0, index[1], 90 if indexed[1] else 0, pads=pads, seed=m)
    run_groupedk(gpu, kind, kind, 264, 256, total, offsets_of(LENGTHS, 3), len(LENGTHS), index[0], 90 if indexed[0] else 0, index[1], 90 if indexed[1] else 0, alpha=-2.0, beta=0.5, pads=(0, 8, 4), seed=9)


# (m, n, lengths of the groups): few tiles with many rows, whose sums are taken in parts of 256 x 256 and of 128 x 128 tiles, or in one of the latter
IN_PARTS = ((264, 264, [700, 0, 333, 1, 65, 5000]), (128, 128, [3000]), (520, 1000, [2100, 2100, 2100, 2100, 2100, 0, 6000, 64]), (100, 300, [0, 0, 1300, 20, 257]), (72, 80, [12000, 1]),
            (520, 264, [40, 100, 3]))


@pytest.mark.parametrize("indexed", ((False, False), (True, True)), ids=str)
@pytest.mark.parametrize("m,n,lengths", IN_PARTS, ids=str)
def test_sums_in_parts(gpu, m, n, lengths, indexed):
    total = sum(lengths) + 5
    rng = np.random.default_rng(total)
    index = [rng.integers(-1, 90, total) if i else None for i in indexed]
    rows = [90 if i else 0 for i in indexed]
    for kind, out, alpha, beta in (("bf16", "f32", 1.0, 0.0), ("f16", "f16", 0.5, -1.0), ("bf16", "bf16", 1.0, 0.0), ("f16", "f32", -1.0, 2.0)):
        run_groupedk(gpu, kind, out, m, n, total, offsets_of(lengths, 3), len(lengths), index[0], rows[0], index[1], rows[1], alpha=alpha, beta=beta, pads=(-m % 8, -n % 8, 4), seed=m)


def test_the_same_bits_of_sums_in_parts(gpu):
    first, second = (run_groupedk(gpu, "bf16", "f32", 256, 256, 9000, offsets_of([4000, 5000]), 2, seed=5) for _ in range(2))
    assert np.array_equal(first.view(np.uint32), second.view(np.uint32))


def test_few_columns_of_a_sum(gpu):
    """Fewer than the eight values that are loaded at once."""
    for m, n in ((1, 7), (7, 1), (8, 7), (7, 200), (200, 3), (9, 9)):
        run_groupedk(gpu, "bf16", "f32", m, n, 150, offsets_of([70, 0, 80]), 3, seed=m)
        run_grouped(gpu, "bf16", "f32", 150, n, 70, offsets_of([70, 0, 80]), 3, layout="row", seed=m)


def put(lib, address, values):
    values = np.ascontiguousarray(values)
    assert lib.skl_hip_memcpy_h2d(address, values.ctypes.data, values.nbytes) == 0


def get(lib, address, shape, dtype):
    out = np.empty(shape, dtype)
    assert lib.skl_hip_memcpy_d2h(out.ctypes.data, address, out.nbytes) == 0
    return out


def test_operands_beyond_four_gib(gpu):
    """Rows of A and C, matrices of B, whose bytes are further than 2^32 from the first; the rest of the memory is NaN."""
    rng = np.random.default_rng(7)
    m, n, k, pitch = 70000, 256, 64, 40000  # 5.6e9 bytes of A, 11.2e9 of C
    whole = lambda shape: gs.bits(rng.integers(-4, 5, shape), "bf16")  # sums of whole numbers: exact  # noqa: E731
    a, c = DeviceBuffer(2 * m * pitch), DeviceBuffer(4 * m * pitch)
    gsb = 1 << 30
    b = DeviceBuffer(2 * (3 * gsb + n * k))
    for buf in (a, b, c):
        gpu.skl_hip_memset(buf, 0xFF, buf.nbytes)
    groups = np.array([0, 3, 69990, 69990, 70000], np.int32)
    o = DeviceBuffer.from_array(groups)
    rows = [0, 1, 2, 3, 255, 256, 60001, 69989, 69990, 69999]
    x, w = whole((len(rows), k)), whole((4, n, k))
    for i, r in enumerate(rows):
        put(gpu, a.offset(2 * r * pitch), x[i])
    for e in range(4):
        put(gpu, b.offset(2 * e * gsb), w[e])
    xv, wv = gs.values(x, "bf16"), gs.values(w, "bf16")
    group_of = lambda r: int(np.searchsorted(groups, r, side="right")) - 1  # noqa: E731
    want = np.stack([xv[i] @ wv[group_of(r)].T for i, r in enumerate(rows)])
    gpu.skl_gemm_grouped_bf16_bf16rc_f32_gfx950(4, o, m, n, k, 1.0, a, pitch, None, 0, b, 1, k, gsb, 0.0, c, pitch)
    assert gpu.skl_hip_synchronize() == 0
    skl_amd.check_error()
    for i, r in enumerate(rows):
        assert np.array_equal(get(gpu, c.offset(4 * r * pitch), (n,), np.float32), want[i]), r
        assert np.isnan(get(gpu, c.offset(4 * (r * pitch + n)), (1,), np.float32))
    # the same rows through an index, the products summed over them, and with another pitch of four bytes
    index = np.array(rows, np.int32)
    oi = DeviceBuffer.from_array(np.searchsorted(index, groups).astype(np.int32))
    di, small = DeviceBuffer.from_array(index), DeviceBuffer(4 * len(rows) * n)
    gpu.skl_gemm_grouped_bf16_bf16rc_f32_gfx950(4, oi, len(rows), n, k, 1.0, a, pitch, di, m, b, 1, k, gsb, 0.0, small, n)
    assert np.array_equal(get(gpu, small.ptr, (len(rows), n), np.float32), want)
    y = whole((len(rows), n))
    dy, sums = DeviceBuffer.from_array(y), DeviceBuffer(4 * 4 * n * k)
    gpu.skl_gemm_groupedk_bf16c_bf16_f32_gfx950(4, oi, n, k, len(rows), 1.0, dy, n, None, 0, a, pitch, di, m, 0.0, sums, k, n * k)
    got = get(gpu, sums.ptr, (4, n, k), np.float32)
    skl_amd.check_error()
    yv = gs.values(y, "bf16")
    for e in range(4):
        mine = [i for i, r in enumerate(rows) if group_of(r) == e]
        assert np.array_equal(got[e], yv[mine].T @ xv[mine])


def test_4_bit_weights_beyond_four_gib(gpu):
    from skl_amd import U4Weights
    rng = np.random.default_rng(8)
    n, k, expert = 48, 256, 10_000_000_000  # 5e9 bytes from one matrix to the next
    expert -= expert % 32
    codes = DeviceBuffer(expert + n * k // 2)
    gpu.skl_hip_memset(codes, 0xFF, codes.nbytes)
    q = rng.integers(0, 16, (3, n, k)).astype(np.uint8)
    for e in range(3):
        put(gpu, codes.offset(e * (expert // 2)), gs.u4_store(q[e], k))
    scales = DeviceBuffer.from_array(gs.bits(np.ones((3, n, 2)), "bf16"))
    a = gs.bits(rng.integers(-4, 5, (5, k)), "bf16")
    da, c, o = DeviceBuffer.from_array(a), DeviceBuffer(4 * 5 * n), DeviceBuffer.from_array(np.array([0, 1, 1, 5], np.int32))
    w = U4Weights(group_k=128, codes=codes, ld=k, expert=expert, scales=scales, zeros=None, ld_scales=2, expert_scales=2 * n)
    gpu.skl_gemm_grouped_bf16_u4c_f32_gfx950(3, o, 5, n, k, 1.0, da, k, None, 0, w, 0.0, c, n)
    got = get(gpu, c.ptr, (5, n), np.float32)
    skl_amd.check_error()
    v = gs.values(a, "bf16")
    assert np.array_equal(got[:1], v[:1] @ (q[0].astype(np.float64) - 8).T) and np.array_equal(got[1:], v[1:] @ (q[2].astype(np.float64) - 8).T)

"""Products grouped by expert - over groups of rows, and summed over them - against their definition in 64 bits, on any layout. The bounds are
those of fp32 sums of exact products (grouped_support.gamma), with half a step of C's type on top."""
import numpy as np
import pytest

import grouped_support as gs
import skl_amd
from skl_amd import DeviceBuffer

pytestmark = pytest.mark.gpu

KINDS = ("bf16", "f16")
NAN = {"bf16": 0x7FC1, "f16": 0x7E01}


def strided(x, pitch, fill, front=0, tail=0):
    """A flat array with the rows of x `pitch` apart, `fill` in between, `front` elements ahead of it."""
    rows, cols = x.shape
    flat = np.full(front + (rows - 1) * pitch + cols + tail if rows else front + tail, fill, x.dtype)
    for i in range(rows):
        flat[front + i * pitch:front + i * pitch + cols] = x[i]
    return flat


def rows_of(flat, rows, cols, pitch, front=0):
    return np.stack([flat[front + i * pitch:front + i * pitch + cols] for i in range(rows)]) if rows else np.zeros((0, cols), flat.dtype)


def split(rng, rows, groups, empty=0.25):
    """Ascending offsets over `rows` rows, some groups empty."""
    shares = rng.random(groups) * (rng.random(groups) >= empty)
    if shares.sum() == 0:
        shares[-1] = 1.0
    return np.concatenate(([0], np.floor(np.cumsum(shares) / shares.sum() * rows + 0.5))).astype(np.int32)


def run_grouped(lib, kind, out, m, n, k, offsets, groups, index=None, a_rows=None, layout="col", alpha=1.0, beta=0.0, seed=0, pads=(0, 0, 0), fronts=(0, 0, 0), mode="device", spoil_c=True):
    """One call on random operands with NaN in everything that is not to be looked at, checked."""
    rng = np.random.default_rng(seed)
    a_count = m if index is None else a_rows
    a = gs.bits(rng.normal(size=(a_count, k)), kind)
    b = [gs.bits(rng.normal(size=(k, n)), kind) for _ in range(groups)]
    old = gs.bits(rng.normal(size=(m, n)), out)
    ranges = gs.cut(offsets, m, groups)
    used = np.zeros(a_count, bool)
    for first, end in ranges:
        at = np.arange(first, end) if index is None else np.asarray(index[first:end], np.int64)
        used[at[(at >= 0) & (at < a_count)]] = True
    a[~used] = NAN[kind]  # rows of A that no group has
    pa, pb, pc = pads
    flat_a = strided(a, k + pa, NAN[kind], fronts[0], 9)
    if layout == "col":
        rsb, csb = 1, k + pb
        flats = [strided(w.T, k + pb, NAN[kind]) for w in b]
    elif layout == "row":
        rsb, csb = n + pb, 1
        flats = [strided(w, n + pb, NAN[kind]) for w in b]
    else:  # no unit stride
        rsb, csb = 3, 3 * k + pb + 1
        flats = []
        for w in b:
            f = np.full((n - 1) * csb + (k - 1) * 3 + 1 if k else 1, NAN[kind], np.uint16)
            for j in range(n):
                f[j * csb:j * csb + 3 * k:3] = w[:, j] if k else 0
            flats.append(f)
    gsb = max(len(f) for f in flats) + pb
    flat_b = np.full(fronts[1] + (groups - 1) * gsb + len(flats[-1]) + 9, NAN[kind], np.uint16)
    for e, f in enumerate(flats):
        flat_b[fronts[1] + e * gsb:fronts[1] + e * gsb + len(f)] = f
    spoil = np.float32(np.nan) if out == "f32" else NAN[out]
    if beta == 0.0 and spoil_c:
        shown = np.full(old.shape, spoil, old.dtype)  # an old C that is not read
    else:
        shown = old
    flat_c = strided(shown, n + pc, spoil, fronts[2], 9)
    item = 4 if out == "f32" else 2
    idx = None if index is None else np.asarray(index, np.int32)
    offs = None if offsets is None else np.asarray(offsets, np.int32)
    entry = getattr(lib, f"skl_gemm_grouped_{kind}_{kind}rc_{out}_gfx950")

    def args(A, I, O, B, C):
        return (groups, O, m, n, k, alpha, A, k + pa, I, a_rows or 0, B, rsb, csb, gsb, beta, C, n + pc)
    if mode == "host":
        got = flat_c.copy()
        entry(*args(flat_a[fronts[0]:], idx, offs, flat_b[fronts[1]:], got[fronts[2]:]))
        skl_amd.check_error()
    else:
        da, db, dc = (DeviceBuffer.from_array(f) for f in (flat_a, flat_b, flat_c))
        di, do = (None if v is None else DeviceBuffer.from_array(v) for v in (idx, offs))
        entry(*args(da.offset(2 * fronts[0]), di, do, db.offset(2 * fronts[1]), dc.offset(item * fronts[2])))
        assert lib.skl_hip_synchronize() == 0
        skl_amd.check_error()
        got = dc.download(flat_c.dtype, flat_c.size)
    clean = a.copy()
    clean[~used] = 0
    want, bound, inside = gs.product(gs.values(clean, kind), [gs.values(w, kind) for w in b], gs.values(old, out), alpha, beta, ranges, index)
    have = rows_of(got, m, n, n + pc, fronts[2])
    raw = have.view(np.uint32 if out == "f32" else np.uint16)
    was = shown.view(np.uint32 if out == "f32" else np.uint16)
    assert np.array_equal(raw[~inside], was[~inside]), "a row in no group was written"
    gaps = np.ones(flat_c.size, bool)
    for i in range(m):
        gaps[fronts[2] + i * (n + pc):fronts[2] + i * (n + pc) + n] = False
    assert np.array_equal(got.view(raw.dtype)[gaps], flat_c.view(raw.dtype)[gaps]), "something beside C was written"
    off = np.abs(gs.values(have, out) - want)[inside]
    limit = gs.rounded(want, bound, out)[inside]
    assert np.all(off <= limit), f"{np.nanmax(off / np.maximum(limit, 1e-300))} of the bound"
    return got


SIZES = [(1, 1, 1, 1), (1, 16, 32, 3), (3, 5, 7, 2), (64, 128, 64, 4), (129, 257, 65, 3), (300, 136, 200, 70), (17, 1000, 513, 5), (700, 384, 320, 6), (513, 264, 1032, 2)]


@pytest.mark.parametrize("layout", ("col", "row", "strided"))
@pytest.mark.parametrize("m,n,k,groups", SIZES)
@pytest.mark.parametrize("kind", KINDS)
def test_grouped_products(gpu, kind, m, n, k, groups, layout):
    rng = np.random.default_rng(m * n + k)
    for out in ("f32", kind):
        run_grouped(gpu, kind, out, m, n, k, split(rng, m, groups), groups, layout=layout, seed=m + n)


@pytest.mark.parametrize("mode", ("host", "device"))
@pytest.mark.parametrize("layout", ("col", "row"))
@pytest.mark.parametrize("out", ("f32", "bf16"))
def test_gathered_rows(gpu, out, layout, mode):
    """The same row many times, rows outside A (zeros), padding at the end."""
    rng = np.random.default_rng(5)
    for m, n, k, groups, a_rows in ((90, 72, 64, 5, 30), (400, 256, 136, 9, 130), (7, 33, 31, 2, 1)):
        index = rng.integers(0, a_rows, m)
        index[rng.random(m) < 0.1] = rng.choice([-1, a_rows, -2 ** 31, 2 ** 31 - 1])
        offsets = split(rng, m - m // 5, groups)
        run_grouped(gpu, "bf16", out, m, n, k, offsets, groups, index=index, a_rows=a_rows, layout=layout, seed=m, mode=mode)


@pytest.mark.parametrize("kind", KINDS)
def test_alpha_beta_and_pitches(gpu, kind):
    rng = np.random.default_rng(8)
    for pads in ((0, 0, 0), (8, 8, 8), (8, 16, 3), (3, 5, 1), (2, 2, 2)):
        for layout in ("col", "row"):
            for out in ("f32", kind):
                for m, n, k in ((200, 136, 96), (150, 130, 72)):
                    run_grouped(gpu, kind, out, m, n, k, split(rng, m, 4), 4, layout=layout, alpha=-1.5, beta=0.75, pads=pads, seed=sum(pads))


@pytest.mark.parametrize("fronts", ((1, 0, 0), (0, 1, 0), (0, 0, 1), (4, 2, 2), (3, 5, 7)))
def test_operands_on_any_boundary(gpu, fronts):
    rng = np.random.default_rng(9)
    for layout in ("col", "row"):
        for out in ("f32", "f16"):
            run_grouped(gpu, "f16", out, 260, 264, 128, split(rng, 260, 3), 3, layout=layout, fronts=fronts, seed=sum(fronts))


def test_no_products_and_no_rows(gpu):
    """k == 0 scales C on the groups' rows; empty lists touch nothing; an A without rows counts as zeros."""
    offsets = np.array([2, 2, 5, 9], np.int32)
    for out in ("f32", "bf16"):
        run_grouped(gpu, "bf16", out, 12, 20, 0, offsets, 3, beta=0.5)
        run_grouped(gpu, "bf16", out, 12, 20, 0, offsets, 3, beta=0.0)
        run_grouped(gpu, "bf16", out, 12, 20, 40, np.zeros(4, np.int32), 3, beta=0.5)
        run_grouped(gpu, "bf16", out, 12, 20, 40, offsets, 3, index=np.zeros(12, np.int32), a_rows=0, beta=0.5)
    gpu.skl_gemm_grouped_bf16_bf16rc_f32_gfx950(3, None, 0, 20, 40, 1.0, None, 40, None, 0, None, 1, 40, 800, 0.0, None, 20)
    gpu.skl_gemm_grouped_bf16_bf16rc_f32_gfx950(0, None, 12, 20, 40, 1.0, None, 40, None, 0, None, 1, 40, 800, 0.0, None, 20)
    skl_amd.check_error()


@pytest.mark.parametrize("m", (1, 130, 600))
def test_one_group_without_offsets(gpu, m):
    for layout in ("col", "row"):
        run_grouped(gpu, "bf16", "bf16", m, 264, 192, None, 1, layout=layout, seed=m)


def test_offsets_are_cut_off(gpu):
    """Offsets below zero and beyond m reach nothing outside C."""
    for offsets in ([-5, 3, 40, 90], [-2 ** 31, 10, 2 ** 31 - 1, 2 ** 31 - 1], [10, 10, 12, 12], [64, 64, 64, 64], [70, 80, 90, 100]):
        for k in (64, 33):
            run_grouped(gpu, "f16", "f32", 64, 136, k, np.array(offsets, np.int64).astype(np.int32), 3, seed=k)


def test_offsets_that_fall_back_write_rows_of_c_alone(gpu):
    """Which rows are written is open then, but none outside C: the elements around it stay."""
    m, n, k, pitch = 300, 264, 64, 270
    rng = np.random.default_rng(1)
    a, b = (DeviceBuffer.from_array(gs.bits(rng.normal(size=s), "bf16")) for s in ((m, k), (3, n, k)))
    fill = np.full(16 + m * pitch + 16, 7.0, np.float32)
    c = DeviceBuffer.from_array(fill)
    for offsets in ([0, 300, 0, 300], [300, 0, 300, 0], [100, 300, 50, 200]):
        o = DeviceBuffer.from_array(np.array(offsets, np.int32))
        gpu.skl_gemm_grouped_bf16_bf16rc_f32_gfx950(3, o, m, n, k, 1.0, a, k, None, 0, b, 1, k, n * k, 0.0, c.offset(64), pitch)
        assert gpu.skl_hip_synchronize() == 0
        skl_amd.check_error()
        got = c.download(np.float32, fill.size)
        assert np.all(got[:16] == 7) and np.all(got[-16:] == 7) and np.all(got[16:16 + m * pitch].reshape(m, pitch)[:, n:] == 7)


def test_infinities_and_nan_stay_in_their_rows(gpu):
    m, n, k = 140, 136, 72
    rng = np.random.default_rng(2)
    av = rng.integers(-4, 5, (m, k)).astype(np.float32)
    bv = rng.integers(1, 5, (2, n, k)).astype(np.float32)
    av[3, 5], av[77, 0], av[139, 71] = np.inf, np.nan, -np.inf
    for kind in KINDS:
        a, b, c = DeviceBuffer.from_array(gs.bits(np.nan_to_num(av, nan=0, posinf=0, neginf=0), kind)), DeviceBuffer.from_array(gs.bits(bv, kind)), DeviceBuffer(4 * m * n)
        special = gs.bits(np.nan_to_num(av, nan=0, posinf=0, neginf=0), kind)
        inf = {"bf16": (0x7F80, 0xFF80), "f16": (0x7C00, 0xFC00)}[kind]
        special[3, 5], special[77, 0], special[139, 71] = inf[0], NAN[kind], inf[1]
        a.upload(special)
        o = DeviceBuffer.from_array(np.array([0, 70, 140], np.int32))
        getattr(gpu, f"skl_gemm_grouped_{kind}_{kind}rc_f32_gfx950")(2, o, m, n, k, 1.0, a, k, None, 0, b, 1, k, n * k, 0.0, c, n)
        assert gpu.skl_hip_synchronize() == 0
        got = c.download(np.float32, m * n).reshape(m, n)
        assert np.all(got[3] == np.inf) and np.all(np.isnan(got[77])) and np.all(got[139] == -np.inf)
        rest = np.ones(m, bool)
        rest[[3, 77, 139]] = False
        want = np.concatenate([av[:70] @ bv[0].T, av[70:] @ bv[1].T])
        assert np.array_equal(got[rest], want[rest])  # whole numbers: exact


def test_beta_zero_as_the_reference_evaluates_it(gpu):
    m, n, k = 130, 24, 32
    a, b = DeviceBuffer.from_array(gs.bits(np.ones((m, k)), "bf16")), DeviceBuffer.from_array(gs.bits(np.ones((n, k)), "bf16"))
    for out, dtype in (("f32", np.float32), ("bf16", np.uint16)):
        old = gs.bits(np.ones((m, n)), out)
        old[5, 6] = np.nan if out == "f32" else 0x7FC0
        for mode in (0, 1):
            c = DeviceBuffer.from_array(old)
            gpu.skl_hip_set_beta_zero_mode(mode)
            try:
                getattr(gpu, f"skl_gemm_grouped_bf16_bf16rc_{out}_gfx950")(1, None, m, n, k, 1.0, a, k, None, 0, b, 1, k, n * k, 0.0, c, n)
            finally:
                gpu.skl_hip_set_beta_zero_mode(0)
            assert gpu.skl_hip_synchronize() == 0
            got = gs.values(c.download(dtype, m * n), out).reshape(m, n)
            assert np.isnan(got[5, 6]) == (mode == 1)
            got[5, 6] = k
            assert np.all(got == k)


# ----------------------------------------------------------------------------------------------------------------------
# sums over groups of rows
# ----------------------------------------------------------------------------------------------------------------------

def run_groupedk(lib, kind, out, m, n, total, offsets, groups, index_a=None, a_rows=0, index_b=None, b_rows=0, alpha=1.0, beta=0.0, seed=0, pads=(0, 0, 0), fronts=(0, 0, 0), mode="device"):
    rng = np.random.default_rng(seed)
    ranges = gs.cut(offsets, total, groups)
    operands, flats, clean = [], [], []
    for cols, index, given, pad, front in ((m, index_a, a_rows, pads[0], fronts[0]), (n, index_b, b_rows, pads[1], fronts[1])):
        count = total if index is None else given
        x = gs.bits(rng.normal(size=(count, cols)), kind)
        used = np.zeros(count, bool)
        for first, end in ranges:
            at = np.arange(first, end) if index is None else np.asarray(index[first:end], np.int64)
            used[at[(at >= 0) & (at < count)]] = True
        x[~used] = NAN[kind]
        operands.append(x)
        flats.append(strided(x, cols + pad, NAN[kind], front, 9))
        x = x.copy()
        x[~used] = 0
        clean.append(gs.values(x, kind))
    old = gs.bits(rng.normal(size=(groups, m, n)), out)
    spoil = np.float32(np.nan) if out == "f32" else NAN[out]
    shown = np.full(old.shape, spoil, old.dtype) if beta == 0.0 else old
    rsc, gsc = n + pads[2], (m - 1) * (n + pads[2]) + n + 3 * pads[2]
    flat_c = np.full(fronts[2] + (groups - 1) * gsc + (m - 1) * rsc + n + 9, spoil, old.dtype)
    mine = np.zeros(flat_c.size, bool)
    for e in range(groups):
        for i in range(m):
            at = fronts[2] + e * gsc + i * rsc
            flat_c[at:at + n] = shown[e, i]
            mine[at:at + n] = True
    entry = getattr(lib, f"skl_gemm_groupedk_{kind}c_{kind}_{out}_gfx950")
    ints = [None if v is None else np.asarray(v, np.int32) for v in (offsets, index_a, index_b)]

    def args(o, a, ia, b, ib, c):
        return (groups, o, m, n, total, alpha, a, m + pads[0], ia, a_rows, b, n + pads[1], ib, b_rows, beta, c, rsc, gsc)
    if mode == "host":
        got = flat_c.copy()
        entry(*args(ints[0], flats[0][fronts[0]:], ints[1], flats[1][fronts[1]:], ints[2], got[fronts[2]:]))
        skl_amd.check_error()
    else:
        da, db, dc = (DeviceBuffer.from_array(f) for f in (*flats, flat_c))
        do, dia, dib = (None if v is None else DeviceBuffer.from_array(v) for v in ints)
        entry(*args(do, da.offset(2 * fronts[0]), dia, db.offset(2 * fronts[1]), dib, dc.offset((4 if out == "f32" else 2) * fronts[2])))
        assert lib.skl_hip_synchronize() == 0
        skl_amd.check_error()
        got = dc.download(flat_c.dtype, flat_c.size)
    want, bound = gs.over(*clean, gs.values(old, out), alpha, beta, ranges, index_a, index_b, total)
    plain = got.view(np.uint32 if out == "f32" else np.uint16)
    assert np.array_equal(plain[~mine], flat_c.view(plain.dtype)[~mine]), "something beside C was written"
    have = np.stack([rows_of(got, m, n, rsc, fronts[2] + e * gsc) for e in range(groups)])
    off, limit = np.abs(gs.values(have, out) - want), gs.rounded(want, bound, out)
    assert np.all(off <= limit), f"{np.nanmax(off / np.maximum(limit, 1e-300))} of the bound"
    return got


@pytest.mark.parametrize("m,n,total,groups", [(1, 1, 1, 1), (5, 3, 9, 4), (64, 128, 200, 3), (136, 264, 333, 5), (129, 65, 1000, 2), (256, 512, 700, 8), (40, 24, 5000, 70)])
@pytest.mark.parametrize("kind", KINDS)
def test_sums_over_groups(gpu, kind, m, n, total, groups):
    rng = np.random.default_rng(m + n)
    for out in ("f32", kind):
        run_groupedk(gpu, kind, out, m, n, total, split(rng, total, groups), groups, seed=total)


@pytest.mark.parametrize("mode", ("host", "device"))
def test_sums_over_gathered_rows(gpu, mode):
    rng = np.random.default_rng(11)
    for m, n, total, groups, a_rows, b_rows in ((72, 136, 300, 5, 90, 50), (264, 256, 500, 3, 500, 1), (9, 31, 40, 2, 7, 8)):
        index = [rng.integers(0, rows, total) for rows in (a_rows, b_rows)]
        for v, rows in zip(index, (a_rows, b_rows)):
            v[rng.random(total) < 0.1] = rng.choice([-1, rows, -2 ** 31, 2 ** 31 - 1])
        offsets = split(rng, total - total // 6, groups)
        for which in ((True, False), (False, True), (True, True)):
            run_groupedk(gpu, "bf16", "f32", m, n, total, offsets, groups, index[0] if which[0] else None, a_rows if which[0] else 0, index[1] if which[1] else None,
                         b_rows if which[1] else 0, seed=m, mode=mode)


def test_sums_alpha_beta_pitches_and_boundaries(gpu):
    rng = np.random.default_rng(12)
    for pads, fronts in (((8, 8, 8), (0, 0, 0)), ((0, 0, 1), (0, 0, 0)), ((3, 1, 2), (1, 3, 5)), ((8, 8, 4), (8, 8, 4))):
        for out in ("f32", "f16"):
            run_groupedk(gpu, "f16", out, 136, 264, 400, split(rng, 400, 4), 4, alpha=-0.5, beta=1.25, pads=pads, fronts=fronts, seed=pads[0])


def test_sums_over_nothing(gpu):
    for out in ("f32", "bf16"):
        for offsets in (np.zeros(4, np.int32), np.array([5, 5, 9, 9], np.int32), np.array([30, 40, 50, 60], np.int32)):
            run_groupedk(gpu, "bf16", out, 20, 40, 12, offsets, 3, beta=0.5)
            run_groupedk(gpu, "bf16", out, 20, 40, 12, offsets, 3)
        run_groupedk(gpu, "bf16", out, 20, 40, 0, np.zeros(4, np.int32), 3, beta=0.5)
        run_groupedk(gpu, "bf16", out, 20, 40, 50, None, 1)


@pytest.mark.parametrize("kind", KINDS)
def test_the_same_bits_on_every_run(gpu, kind):
    rng = np.random.default_rng(13)
    offsets = split(rng, 700, 9)
    first = [run_grouped(gpu, kind, "f32", 700, 264, 520, offsets, 9), run_groupedk(gpu, kind, "f32", 264, 136, 700, offsets, 9)]
    for _ in range(3):
        again = [run_grouped(gpu, kind, "f32", 700, 264, 520, offsets, 9), run_groupedk(gpu, kind, "f32", 264, 136, 700, offsets, 9)]
        for x, y in zip(first, again):
            assert np.array_equal(x.view(np.uint32), y.view(np.uint32))

"""Products with integer 4-bit weights in groups against their definition in 64 bits. Products with q - z are exact; their sums within a group are fp32 sums of k
values in any order, each times its scale and added up: one more rounding per group and one for the scale, within gamma(k) of the sum of magnitudes with two more steps."""
import numpy as np
import pytest

import grouped_support as gs
import skl_amd
from skl_amd import DeviceBuffer, U4Weights
from test_gpu_gemm_grouped import NAN, rows_of, split, strided

pytestmark = pytest.mark.gpu


def run_u4(lib, kind, out, m, n, k, group_k, offsets=None, groups=1, zeros="some", index=None, a_rows=0, alpha=1.0, beta=0.0, seed=0, pads=(0, 0, 0), fronts=(0, 0), mode="device"):
    rng = np.random.default_rng(seed)
    count = m if index is None else a_rows
    blocks = -(-k // group_k)
    a = gs.bits(rng.normal(size=(count, k)), kind)
    ranges = gs.cut(offsets, m, groups)
    used = np.zeros(count, bool)
    for first, end in ranges:
        at = np.arange(first, end) if index is None else np.asarray(index[first:end], np.int64)
        used[at[(at >= 0) & (at < count)]] = True
    a[~used] = NAN[kind]
    q = rng.integers(0, 16, (groups, n, k)).astype(np.uint8)
    ld, ld_scales = k + k % 2 + 2 * pads[1], blocks + pads[1]
    expert, expert_scales = (n - 1) * ld + k + k % 2 + 4 * pads[1], (n - 1) * ld_scales + blocks + pads[1]
    scales = gs.bits(rng.uniform(0.01, 0.1, (groups, n, blocks)) * rng.choice([-1, 1], (groups, n, blocks)), kind)
    z = {"some": lambda: rng.integers(0, 16, (groups, n, blocks)), "far": lambda: rng.integers(0, 256, (groups, n, blocks)), None: lambda: None}[zeros]()
    codes = np.full(fronts[1] + (groups - 1) * (expert // 2) + (n - 1) * (ld // 2) + (k + 1) // 2 + 9, 0xA5, np.uint8)
    sc = np.full((groups - 1) * expert_scales + (n - 1) * ld_scales + blocks, NAN[kind], np.uint16)
    zs = np.full(sc.size, 201, np.uint8)
    for e in range(groups):
        f = gs.u4_store(q[e], ld)
        codes[fronts[1] + e * (expert // 2):][:len(f)] = f
        for j in range(n):
            at = e * expert_scales + j * ld_scales
            sc[at:at + blocks] = scales[e, j]
            if z is not None:
                zs[at:at + blocks] = z[e, j]
    old = gs.bits(rng.normal(size=(m, n)), out)
    spoil = np.float32(np.nan) if out == "f32" else NAN[out]
    shown = np.full(old.shape, spoil, old.dtype) if beta == 0.0 else old
    flat_a, flat_c = strided(a, k + pads[0], NAN[kind], fronts[0], 9), strided(shown, n + pads[2], spoil, 0, 9)
    entry = getattr(lib, f"skl_gemm_grouped_{kind}_u4c_{out}_gfx950")
    ints = [None if v is None else np.asarray(v, np.int32) for v in (offsets, index)]

    def call(o, i, A, C, co, s, zz):
        w = U4Weights(group_k=group_k, codes=co, ld=ld, expert=expert, scales=s, zeros=zz, ld_scales=ld_scales, expert_scales=expert_scales)
        entry(groups, o, m, n, k, alpha, A, k + pads[0], i, a_rows, w, beta, C, n + pads[2])
    if mode == "host":
        got = flat_c.copy()
        call(*ints, flat_a[fronts[0]:], got, codes[fronts[1]:], sc, zs if z is not None else None)
        skl_amd.check_error()
    else:
        bufs = [None if v is None else DeviceBuffer.from_array(v) for v in (*ints, flat_a, flat_c, codes, sc, zs if z is not None else None)]
        call(bufs[0], bufs[1], bufs[2].offset(2 * fronts[0]), bufs[3], bufs[4].offset(fronts[1]), bufs[5], bufs[6])
        assert lib.skl_hip_synchronize() == 0
        skl_amd.check_error()
        got = bufs[3].download(flat_c.dtype, flat_c.size)
    clean = a.copy()
    clean[~used] = 0
    w = [gs.u4_weights(q[e], gs.values(scales[e], kind), None if z is None else z[e], group_k) for e in range(groups)]
    want, bound, inside = gs.product(gs.values(clean, kind), w, gs.values(old, out), alpha, beta, ranges, index)
    bound = bound * (gs.gamma(k + 2) / gs.gamma(k))
    have = rows_of(got, m, n, n + pads[2])
    raw, was = (v.view(np.uint32 if out == "f32" else np.uint16) for v in (have, shown))
    assert np.array_equal(raw[~inside], was[~inside]), "a row in no group was written"
    off, limit = np.abs(gs.values(have, out) - want)[inside], gs.rounded(want, bound, out)[inside]
    assert np.all(off <= limit), f"{np.nanmax(off / np.maximum(limit, 1e-300))} of the bound"
    return got


@pytest.mark.parametrize("k,group_k", [(32, 32), (64, 32), (256, 64), (256, 128), (448, 128), (1024, 256), (4096, 128), (2048, 4096), (2304, 32)])
@pytest.mark.parametrize("kind", ("bf16", "f16"))
def test_an_ordinary_layer(gpu, kind, k, group_k):
    for m, n in ((1, 64), (1, 1000), (3, 257), (16, 48), (17, 128), (70, 40)):
        for zeros in ("some", None):
            run_u4(gpu, kind, "f32" if m != 3 else kind, m, n, k, group_k, zeros=zeros, seed=m + n)


@pytest.mark.parametrize("k,group_k", [(1, 32), (7, 7), (33, 32), (250, 64), (2080, 96)])
def test_any_k(gpu, k, group_k):
    for m, n in ((1, 5), (18, 130)):
        run_u4(gpu, "bf16", "f32", m, n, k, group_k, seed=k)
        run_u4(gpu, "f16", "f16", m, n, k, group_k, zeros=None, seed=k)


@pytest.mark.parametrize("mode", ("host", "device"))
@pytest.mark.parametrize("kind", ("bf16", "f16"))
def test_experts(gpu, kind, mode):
    rng = np.random.default_rng(4)
    for m, n, k, group_k, groups, tokens in ((32, 136, 256, 64, 12, 8), (8, 64, 512, 128, 40, 1), (200, 72, 96, 32, 3, 100)):
        index = rng.integers(0, tokens, m)
        index[rng.random(m) < 0.1] = -1
        run_u4(gpu, kind, kind, m, n, k, group_k, split(rng, m - m // 8, groups), groups, index=index, a_rows=tokens, seed=m, mode=mode)


@pytest.mark.parametrize("kind", ("bf16", "f16"))
def test_zero_points_alpha_beta_pitches_and_boundaries(gpu, kind):
    for pads, fronts in (((0, 0, 0), (0, 0)), ((8, 32, 8), (8, 16)), ((1, 1, 1), (1, 1)), ((8, 16, 0), (0, 0)), ((0, 0, 0), (0, 1)), ((0, 0, 0), (4, 0))):
        for zeros in ("far", "some", None):
            run_u4(gpu, kind, "f32", 5, 72, 256, 64, zeros=zeros, alpha=-2.0, beta=0.5, pads=pads, fronts=fronts, seed=3)
            run_u4(gpu, kind, kind, 18, 72, 256, 128, np.array([1, 7, 7, 18]), 3, zeros=zeros, alpha=0.5, beta=-1.0, pads=pads, fronts=fronts, seed=4)


def test_nothing_to_multiply(gpu):
    run_u4(gpu, "bf16", "f32", 4, 24, 64, 32, np.zeros(3, np.int32), 2, beta=0.5)
    run_u4(gpu, "bf16", "f32", 4, 24, 64, 32, np.array([0, 2, 4]), 2, index=np.zeros(4), a_rows=0, beta=0.5)
    c = DeviceBuffer.from_array(np.full(96, 3.0, np.float32))
    gpu.skl_gemm_grouped_bf16_u4c_f32_gfx950(1, None, 4, 24, 0, 1.0, None, 0, None, 0, None, 0.5, c, 24)
    assert gpu.skl_hip_synchronize() == 0
    skl_amd.check_error()
    assert np.all(c.download(np.float32, 96) == 1.5)


def test_special_values_of_a(gpu):
    """Infinities and NaN stay in their rows and come out as the products make them; the largest numbers do not overflow on the way."""
    n, k = 40, 64
    q = np.full((n, k), 11, np.uint8)
    q[:, 0] = 8
    q[1::2, 1] = 5
    scale = 2.0 ** -6
    for kind, inf, big in (("bf16", 0x7F80, 0x7F7F), ("f16", 0x7C00, 0x7BFF)):
        a = gs.bits(np.ones((5, k)), kind)
        a[1, 1], a[2, 3], a[3, 0] = inf, NAN[kind], inf
        a[4] = 0
        a[4, 1] = big
        bufs = [DeviceBuffer.from_array(v) for v in (a, gs.u4_store(q, k), gs.bits(np.full((n, 2), scale), kind))]
        c = DeviceBuffer(4 * 5 * n)
        w = U4Weights(group_k=32, codes=bufs[1], ld=k, expert=0, scales=bufs[2], zeros=None, ld_scales=2, expert_scales=0)
        getattr(gpu, f"skl_gemm_grouped_{kind}_u4c_f32_gfx950")(1, None, 5, n, k, 1.0, bufs[0], k, None, 0, w, 0.0, c, n)
        assert gpu.skl_hip_synchronize() == 0
        got = c.download(np.float32, 5 * n).reshape(5, n)
        sign = np.where(np.arange(n) % 2, -1.0, 1.0)
        assert np.array_equal(got[0], (q.astype(np.float64) - 8).sum(axis=1) * scale)
        assert np.array_equal(got[1], np.inf * sign)
        assert np.all(np.isnan(got[2])) and np.all(np.isnan(got[3]))  # infinity times zero
        largest = float(gs.values(np.array([big], np.uint16), kind)[0])
        if kind == "f16":  # (3 times the largest bf16 number is beyond fp32)
            assert np.array_equal(got[4], sign * 3 * largest * scale)
        else:
            assert np.array_equal(got[4], np.inf * sign)


def test_the_same_bits_on_every_run(gpu):
    first = run_u4(gpu, "bf16", "f32", 7, 2000, 4096, 128, seed=1)
    for _ in range(3):
        assert np.array_equal(first.view(np.uint32), run_u4(gpu, "bf16", "f32", 7, 2000, 4096, 128, seed=1).view(np.uint32))


@pytest.mark.parametrize("k,group_k", [(96, 32), (160, 32), (192, 64), (1120, 32), (2112, 64), (40, 64)])
@pytest.mark.parametrize("m", (1, 3, 20))
def test_an_infinite_scale_at_the_end(gpu, m, k, group_k):
    """The last group's scale is infinite and its sums are not zero: infinities of their sign, as the definition has it - nothing behind k joins in."""
    n, blocks = 33, -(-k // group_k)
    a = gs.bits(np.ones((m, k)), "bf16")
    q = np.full((n, k), 11, np.uint8)
    q[1::2] = 3
    scales = np.ones((n, blocks), np.float32)
    scales[:, -1] = np.inf
    bufs = [DeviceBuffer.from_array(v) for v in (a, gs.u4_store(q, k), gs.bits(scales, "bf16"))]
    c = DeviceBuffer(4 * m * n)
    w = U4Weights(group_k=group_k, codes=bufs[1], ld=k, expert=0, scales=bufs[2], zeros=None, ld_scales=blocks, expert_scales=0)
    gpu.skl_gemm_grouped_bf16_u4c_f32_gfx950(1, None, m, n, k, 1.0, bufs[0], k, None, 0, w, 0.0, c, n)
    got = c.download(np.float32).reshape(m, n)
    skl_amd.check_error()
    assert np.all(got[:, 0::2] == np.inf) and np.all(got[:, 1::2] == -np.inf)


@pytest.mark.parametrize("m,n,groups", [(1, 10300, 1), (3, 8300, 1), (4, 520, 16), (40, 400, 40), (200, 1100, 64), (30, 10300, 1), (70, 5200, 2)])
@pytest.mark.parametrize("k,group_k,zeros", [(544, 32, "some"), (1600, 64, None), (1184, 2000, "far"), (1280, 128, "some")])
def test_many_workgroups(gpu, m, n, groups, k, group_k, zeros):
    """Sizes at which four waves, not eight, share a column's k."""
    rng = np.random.default_rng(m + n)
    offsets = None if groups == 1 else split(rng, m, groups)
    run_u4(gpu, "f16" if k == 1600 else "bf16", "f32", m, n, k, group_k, offsets=offsets, groups=groups, zeros=zeros, seed=n)

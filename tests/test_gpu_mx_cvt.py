"""Conversions to and from MXFP4 on the GPU: every byte as the definition has it, over both source types, rows and columns, odd lengths and
distances, and the values where a rounding or a scale changes."""
import numpy as np
import pytest

import mx_support as mx
import skl_amd
from gpu_support import MODES, _finish
from skl_amd import DeviceBuffer

pytestmark = pytest.mark.gpu


def call(lib, mode, name, build, arrays, outputs):
    """Runs an entry point on host arrays or device copies; returns the arrays named in `outputs` afterwards."""
    if mode == "host":
        arrays = [a.copy() for a in arrays]
        getattr(lib, name)(*build(*arrays))
        skl_amd.check_error()
        return [arrays[i] for i in outputs]
    bufs = [DeviceBuffer.from_array(a) for a in arrays]
    getattr(lib, name)(*build(*bufs))
    _finish(lib)
    got = [bufs[i].download(arrays[i].dtype, arrays[i].size) for i in outputs]
    for b in bufs:
        b.free()
    return got


def quantise(lib, mode, x, rs, cs, m, k, ld, lds, src):
    """x: flat array of fp32, or of bf16 bits."""
    dst, sc = np.full((m - 1) * (ld // 2) + (k + 1) // 2, 0xA5, np.uint8), np.full((m - 1) * lds + -(-k // 32), 0xA5, np.uint8)
    return call(lib, mode, f"skl_cvt_{src}rc_mxf4e2m1_gfx950", lambda x_, d_, s_: (m, k, x_, rs, cs, d_, ld, s_, lds), [x, dst, sc], (1, 2))


def check(lib, mode, x, rs, cs, m, k, ld, lds, src):
    at = np.arange(m)[:, None] * rs + np.arange(k)[None, :] * cs
    code, scales = mx.quantise((mx.of_bf16(x) if src == "bf16" else x)[at])
    want, want_s = mx.store(code, scales, ld, lds)
    if k % 2:  # the half byte behind an odd row is written as zero
        for i in range(m):
            want[i * (ld // 2) + k // 2] &= 15
    got, got_s = quantise(lib, mode, x, rs, cs, m, k, ld, lds, src)
    assert np.array_equal(got_s, want_s), (np.nonzero(got_s != want_s)[0][:8], got_s[got_s != want_s][:8], want_s[got_s != want_s][:8])
    assert np.array_equal(got, want), (np.nonzero(got != want)[0][:8], got[got != want][:8], want[got != want][:8])


def source(rng, n, src, spread=12):
    x = (rng.normal(size=n) * np.exp2(rng.integers(-spread, spread + 1, size=n))).astype(np.float32)
    return mx.to_bf16(x) if src == "bf16" else x


SHAPES = ((1, 1), (1, 32), (3, 31), (2, 33), (5, 64), (16, 4096), (7, 1000), (1, 257), (130, 96), (129, 513), (33, 255))


@pytest.mark.parametrize("src", ("bf16", "f32"))
@pytest.mark.parametrize("m,k", SHAPES)
def test_rows(gpu, src, m, k):
    rng = np.random.default_rng(m * 1000 + k)
    for mode in MODES:
        for extra, ld, lds in ((0, k + k % 2, -(-k // 32)), (3, k + k % 2 + 6, -(-k // 32) + 3)):
            check(gpu, mode, source(rng, m * (k + extra), src), k + extra, 1, m, k, ld, lds, src)


@pytest.mark.parametrize("src", ("bf16", "f32"))
@pytest.mark.parametrize("m,k", SHAPES)
def test_columns(gpu, src, m, k):
    """The rows of the result are the columns of a k x m matrix."""
    rng = np.random.default_rng(m * 1000 + k + 1)
    for mode in MODES:
        for extra, ld, lds in ((0, k + k % 2, -(-k // 32)), (5, k + k % 2 + 2, -(-k // 32) + 1)):
            check(gpu, mode, source(rng, k * (m + extra), src), 1, m + extra, m, k, ld, lds, src)


@pytest.mark.parametrize("src", ("bf16", "f32"))
def test_any_strides(gpu, src):
    rng = np.random.default_rng(5)
    check(gpu, "device", source(rng, 40000, src), 211, 3, 9, 70, 76, 4, src)
    check(gpu, "device", source(rng, 40000, src), 2, 50, 21, 67, 68, 3, src)


def test_many_rows_of_one_block(gpu):
    """More than the workgroups of one round, every row its own scale."""
    rng = np.random.default_rng(9)
    check(gpu, "device", source(rng, 150000 * 32, "bf16"), 32, 1, 150000, 32, 32, 1, "bf16")


@pytest.mark.parametrize("src", ("bf16", "f32"))
def test_every_exponent_and_the_values_beside_a_midpoint(gpu, src):
    """Each block's largest magnitude is 2^e to just under 2^(e + 1) for every e, subnormal ones included; the others are the E2M1 values, the
    midpoints between them and their neighbours in the source's format, at that block's scale."""
    points = np.array([0.25, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 3.0, 3.5, 4.0, 5.0, 6.0, 7.0])
    rows = []
    for e in range(-149, 128):
        s = max(e - 2, -126)
        for top in (1.0, 1.25, 1.5, 1.75, 1.9921875):
            row = np.zeros(64, np.float32)
            around = np.ldexp(points, s).astype(np.float32)
            around = around[np.abs(around) <= np.ldexp(top, e)]
            beside = np.concatenate([around, np.nextafter(around, np.float32(np.inf)), np.nextafter(around, np.float32(0))])
            beside = beside[beside <= np.ldexp(np.float64(top), e)][:63] * np.where(np.arange(min(63, (beside <= np.ldexp(np.float64(top), e)).sum())) % 3 == 0, -1, 1)
            both = np.concatenate([beside, np.zeros(62 - len(beside[:62]), np.float32)])[:62].astype(np.float32)
            row[:31], row[32:63] = both[:31], both[31:]
            row[31] = row[63] = np.float32(np.ldexp(top, e))
            rows.append(row)
    x = np.array(rows, np.float32)
    if src == "bf16":
        x = mx.to_bf16(x)
    m, k = x.shape
    check(gpu, "device", x.ravel(), k, 1, m, k, k, 2, src)
    check(gpu, "device", np.ascontiguousarray(x.T).ravel(), 1, m, m, k, k, 2, src)


@pytest.mark.parametrize("across", (False, True))
@pytest.mark.parametrize("src", ("bf16", "f32"))
def test_blocks_that_are_not_numbers(gpu, src, across):
    """A NaN or an infinity anywhere takes its block and no other; zeros, of either sign, and blocks of them."""
    rng = np.random.default_rng(3)
    x = rng.normal(size=(160, 96)).astype(np.float32)
    bad = [np.nan, np.inf, -np.inf]
    for i in range(0, 96):
        x[i, i] = bad[i % 3]
    x[100:110, 32:64] = 0.0
    x[110:120, 32:64] = -0.0
    x[120, 3], x[121, 4] = 0.0, -0.0
    x[130:140] = np.float32(2.0 ** -140)  # far below the smallest scale
    flat = (x.T if across else x).ravel().copy()
    if src == "bf16":
        flat = (flat.view(np.uint32) >> 16).astype(np.uint16)  # the upper half keeps NaN and infinity what they are
    check(gpu, "device", flat, *((1, 160) if across else (96, 1)), 160, 96, 96, 3, src)


@pytest.mark.parametrize("dst", ("bf16", "f32"))
@pytest.mark.parametrize("m,k,ld,lds,rs,cs", ((1, 1, 2, 1, 1, 1), (3, 31, 34, 2, 33, 1), (5, 4096, 4096, 128, 4096, 1), (7, 1001, 1010, 40, 1003, 1),
                                             (40, 66, 66, 3, 1, 45), (9, 70, 72, 3, 150, 2)))
def test_back(gpu, dst, m, k, ld, lds, rs, cs):
    """Every code with every scale byte, 0 and 255 among them."""
    rng = np.random.default_rng(k)
    code = rng.integers(0, 16, size=(m, k), dtype=np.uint8)
    scales = rng.integers(0, 256, size=(m, -(-k // 32)), dtype=np.uint8)
    scales.ravel()[:4] = (0, 255, 1, 254)[:scales.size]
    flat, sc = mx.store(code, scales, ld, lds)
    with np.errstate(over="ignore"):
        want = mx.values(code, scales).astype(np.float32)  # 4 and 6 times 2^127 are beyond fp32: infinite
    at = np.arange(m)[:, None] * rs + np.arange(k)[None, :] * cs
    whole = np.full(at.max() + 4, 7.0, np.float32)
    if dst == "bf16":
        whole = mx.to_bf16(whole)
    for mode in MODES:
        got, = call(gpu, mode, f"skl_cvt_mxf4e2m1_{dst}rc_gfx950", lambda s_, c_, d_: (m, k, s_, ld, c_, lds, d_, rs, cs), [flat, sc, whole], (2,))
        v = mx.of_bf16(got) if dst == "bf16" else got
        assert np.array_equal(np.isnan(v[at]), np.isnan(want))
        ok = ~np.isnan(want)
        assert np.array_equal(v[at][ok].view(np.uint32), want[ok].view(np.uint32))
        rest = np.ones(whole.size, bool)
        rest[at.ravel()] = False
        assert np.array_equal(got[rest], whole[rest])


def test_refusals_and_empty_calls(gpu):
    x, d, s = np.ones(64, np.float32), np.full(64, 9, np.uint8), np.full(8, 9, np.uint8)
    refused = [(2, 32, x, 32, 1, d, 31, s, 1), (2, 32, x, 32, 1, d, 30, s, 1), (2, 64, x, 32, 1, d, 64, s, 1), (1, 32, None, 32, 1, d, 32, s, 1)]
    for args in refused:
        gpu.skl_cvt_f32rc_mxf4e2m1_gfx950(*args)
        assert gpu.skl_hip_last_error() == -2, args
    gpu.skl_cvt_mxf4e2m1_f32rc_gfx950(2, 32, d, 33, s, 1, x, 32, 1)
    assert gpu.skl_hip_last_error() == -2
    dev = DeviceBuffer.from_array(x)
    gpu.skl_cvt_f32rc_mxf4e2m1_gfx950(1, 32, dev, 32, 1, d, 32, s, 1)
    assert gpu.skl_hip_last_error() == -1  # device and host memory in one call
    for m, k in ((0, 32), (2, 0)):
        gpu.skl_cvt_f32rc_mxf4e2m1_gfx950(m, k, x, 32, 1, d, 32, s, 1)
        gpu.skl_cvt_mxf4e2m1_f32rc_gfx950(m, k, d, 32, s, 1, x, 32, 1)
        assert gpu.skl_hip_last_error() == 0
    assert (d == 9).all() and (s == 9).all() and (x == 1).all()

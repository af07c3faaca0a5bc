"""Products of two MXFP4 matrices on the GPU, inside the bound of an fp32 sum of exact products and, where every partial sum is a number of
fp32, exact."""
import numpy as np
import pytest

import mx_support as mx
import skl_amd
from gpu_support import MODES, _finish
from skl_amd import DeviceBuffer

pytestmark = pytest.mark.gpu

STEM = "skl_gemm_mxf4e2m1r_mxf4e2m1c_f32rc_gfx950"


def operand(rng, rows, k, ld=None, lds=None, low=121, high=134):
    """(codes, scale bytes, flat arrays, ld, lds)"""
    code = rng.integers(0, 16, size=(rows, k), dtype=np.uint8)
    scales = rng.integers(low, high, size=(rows, -(-k // 32)), dtype=np.uint8)
    ld = k + k % 2 if ld is None else ld
    lds = scales.shape[1] if lds is None else lds
    return (code, scales, *mx.store(code, scales, ld, lds, fill=0xFF), ld, lds)


def run(lib, mode, a, b, k, alpha, beta, c, m, n, rsc, csc):
    def args(fa, sa, fb, sb, c_):
        return (m, n, k, alpha, fa, a[4], sa, a[5], fb, b[4], sb, b[5], beta, c_, rsc, csc)
    if mode == "host":
        out = c.copy()
        getattr(lib, STEM)(*args(a[2], a[3], b[2], b[3], out))
        skl_amd.check_error()
        return out
    bufs = [DeviceBuffer.from_array(v) for v in (a[2], a[3], b[2], b[3], c)]
    getattr(lib, STEM)(*args(*bufs))
    _finish(lib)
    out = bufs[4].download(np.float32, c.size)
    for buf in bufs:
        buf.free()
    return out


def check(lib, mode, rng, m, n, k, alpha=1.0, beta=0.0, rsc=None, csc=1, **layout):
    a = operand(rng, m, k, layout.get("lda"), layout.get("lsa"))
    b = operand(rng, n, k, layout.get("ldb"), layout.get("lsb"))
    rsc = n if rsc is None else rsc
    at = np.arange(m)[:, None] * rsc + np.arange(n)[None, :] * csc
    c = rng.normal(size=at.max() + 3).astype(np.float32)
    want, bound = mx.product_bound(mx.values(a[0], a[1]), mx.values(b[0], b[1]), alpha, beta, c[at].astype(np.float64))
    got = run(lib, mode, a, b, k, alpha, beta, c, m, n, rsc, csc)
    err = np.abs(got[at] - want)
    assert np.all(err <= bound + np.abs(want) * 2.0 ** -22 + 1e-30), (m, n, k, float((err / (bound + 1e-30)).max()))
    rest = np.ones(c.size, bool)
    rest[at.ravel()] = False
    assert np.array_equal(got[rest], c[rest]), "elements outside C were written"
    again = run(lib, mode, a, b, k, alpha, beta, c, m, n, rsc, csc)
    assert np.array_equal(got.view(np.uint32), again.view(np.uint32)), "another result on the second run"


# whole tiles and ragged ones of every kernel, K of one value, of a block, off blocks and chunks, rows off every alignment
SHAPES = ((1, 1, 1), (1, 33, 32), (2, 64, 64), (5, 300, 100), (16, 512, 4096), (17, 130, 513), (31, 1, 700), (33, 65, 31), (64, 64, 256), (65, 129, 288),
          (100, 200, 1000), (128, 128, 512), (130, 257, 2049), (512, 512, 512), (300, 700, 770), (1, 4096, 2080), (48, 1024, 11008), (16, 4100, 256), (17, 8200, 544), (64, 12300, 1024), (3, 9000, 4128),
          (40, 12000, 8192), (64, 64, 14336), (200, 190, 6000))


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_products(gpu, mode, m, n, k):
    rng = np.random.default_rng(m + 7 * n + 11 * k)
    check(gpu, mode, rng, m, n, k)
    check(gpu, mode, rng, m, n, k, alpha=1.5, beta=-0.5, rsc=n + 3)


@pytest.mark.parametrize("m,n,k,layout", (
    (40, 70, 96, dict(lda=128, lsa=7, ldb=110, lsb=5)), (40, 70, 512, dict(lda=512, lsa=16, ldb=544, lsb=17)), (20, 50, 97, dict(lda=98, lsa=4, ldb=102, lsb=5)),
    (3, 500, 1024, dict(lda=1026, lsa=33, ldb=1056, lsb=40)), (200, 300, 768, dict(lda=776, lsa=24, ldb=784, lsb=25))))
def test_distances_off_every_alignment(gpu, m, n, k, layout):
    check(gpu, "device", np.random.default_rng(k), m, n, k, **layout)


@pytest.mark.parametrize("m,n,k", ((70, 90, 256), (8, 200, 512), (300, 260, 320), (1500, 1501, 256)))
def test_c_by_columns_and_with_gaps(gpu, m, n, k):
    rng = np.random.default_rng(m)
    check(gpu, "device", rng, m, n, k, rsc=1, csc=m + 2)
    check(gpu, "device", rng, m, n, k, alpha=2.0, beta=1.0, rsc=1, csc=m)
    check(gpu, "device", rng, m, n, k, rsc=2 * n + 5, csc=2)


@pytest.mark.parametrize("m,n,k,ld", ((2048, 2304, 512, None), (1300, 3400, 300, None), (3500, 4100, 1056, None), (1500, 1472, 257, None), (1409, 1500, 4133, None),
                                      (2048, 4100, 31, None), (2040, 4097, 1315, None), (2049, 6300, 345, 348), (3400, 4097, 64, 66), (3329, 4100, 2049, 2056),
                                      (1500, 1500, 1024, 1024), (2048, 4096, 1536, 1536), (3328, 4096, 512, 520), (1500, 1500, 2047, None)))
def test_large_tiles_are_exact(gpu, m, n, k, ld):
    """One scale everywhere: every partial sum is a multiple of a quarter below 2^24 quarters. Each tile size; K below a block, of one chunk, of several, off blocks
    and chunks; rows that loads to LDS read and rows that are copied."""
    rng = np.random.default_rng(k)
    a, b = operand(rng, m, k, ld, low=127, high=128), operand(rng, n, k, ld, low=127, high=128)
    c = np.full(m * n, np.nan, np.float32)
    got = run(gpu, "device", a, b, k, 1.0, 0.0, c, m, n, n, 1).reshape(m, n)
    want = (mx.values(a[0], a[1]).astype(np.float32) @ mx.values(b[0], b[1]).astype(np.float32).T)  # exact in fp32 for the same reason
    assert np.array_equal(got, want)


@pytest.mark.parametrize("m,n,k", ((16, 96, 640), (70, 40, 640), (300, 4096, 640), (1500, 1500, 1600), (2048, 4096, 2048), (3500, 4096, 1632)))
def test_every_value_and_scale_is_read_back(gpu, m, n, k):
    """Rows of A with a single one read single columns of B, each value times its own block's scale; every scale byte but 255."""
    rng = np.random.default_rng(m)
    b = operand(rng, n, k, low=0, high=255)
    code = np.zeros((m, k), np.uint8)
    pos = (np.arange(m) * 37) % k
    code[np.arange(m), pos] = 2  # 1.0
    scales = np.full((m, k // 32), 127, np.uint8)
    a = (code, scales, *mx.store(code, scales, k, k // 32), k, k // 32)
    got = run(gpu, "device", a, b, k, 1.0, 0.0, np.zeros(m * n, np.float32), m, n, n, 1).reshape(m, n)
    with np.errstate(over="ignore"):
        want = mx.values(b[0], b[1])[:, pos].T.astype(np.float32)
    ok = np.isfinite(want) & ((np.abs(want) >= 2.0 ** -126) | (want == 0))  # the matrix cores' results are normal numbers
    assert np.array_equal(got[ok], want[ok])


def test_scales_of_nan(gpu):
    """A block whose scale byte is 255 makes NaN of its row of C, in A and in B, wherever in K it lies, and of nothing else."""
    rng = np.random.default_rng(4)
    for m, n, k in ((5, 90, 352), (150, 130, 352), (1500, 1500, 352)):
        a, b = operand(rng, m, k), operand(rng, n, k)
        for op, row, block in ((a, 3, 10), (b, 88, 0)):
            op[1][row, block] = 255
            op[3][row * op[5] + block] = 255
        got = run(gpu, "device", a, b, k, 1.0, 0.0, np.zeros(m * n, np.float32), m, n, n, 1).reshape(m, n)
        want = np.zeros((m, n), bool)
        want[3] = True
        want[:, 88] = True
        assert np.array_equal(np.isnan(got), want)


def test_beta_zero_and_empty_sums(gpu):
    rng = np.random.default_rng(8)
    m, n, k = 40, 50, 64
    a, b = operand(rng, m, k), operand(rng, n, k)
    c = np.full(m * n, np.nan, np.float32)
    assert np.isfinite(run(gpu, "device", a, b, k, 1.0, 0.0, c, m, n, n, 1)).all()  # an old C is overwritten
    gpu.skl_hip_set_beta_zero_mode(1)
    try:
        assert np.isnan(run(gpu, "device", a, b, k, 1.0, 0.0, c, m, n, n, 1)).all()  # 0 * NaN
    finally:
        gpu.skl_hip_set_beta_zero_mode(0)
    c = rng.normal(size=m * n).astype(np.float32)
    for mode in MODES:
        assert np.array_equal(run(gpu, mode, a, b, 0, 1.0, 2.0, c, m, n, n, 1), 2 * c)  # k == 0: C = beta C
    kept = c.copy()
    gpu.skl_gemm_mxf4e2m1r_mxf4e2m1c_f32rc_gfx950(0, n, k, 1.0, a[2], k, a[3], 2, b[2], k, b[3], 2, 0.0, c, n, 1)
    gpu.skl_gemm_mxf4e2m1r_mxf4e2m1c_f32rc_gfx950(m, 0, k, 1.0, a[2], k, a[3], 2, b[2], k, b[3], 2, 0.0, c, n, 1)
    assert gpu.skl_hip_last_error() == 0 and np.array_equal(c, kept)


def test_negative_zero_products_take_the_old_sign(gpu):
    """beta == 0: where alpha times the product is a zero, the old C's sign decides as in the reference's 0 * c + x."""
    rng = np.random.default_rng(8)
    m, n, k = 20, 140, 64
    a, b = operand(rng, m, k), operand(rng, n, k)
    a[2][:] = 0
    c = np.where(rng.random(m * n) < 0.5, -1.0, 1.0).astype(np.float32)
    got = run(gpu, "device", a, b, k, -1.0, 0.0, c, m, n, n, 1)
    assert np.array_equal(got.view(np.uint32), (np.float32(0) * c + np.float32(-1) * np.zeros_like(c)).view(np.uint32))


def test_refusals(gpu):
    a = np.zeros(4096, np.uint8)
    c = np.full(64, 3.0, np.float32)
    for lda, lsa, ldb, lsb in ((63, 2, 64, 2), (62, 2, 64, 2), (64, 1, 64, 2), (64, 2, 65, 2), (64, 2, 60, 2), (64, 2, 64, 1)):
        gpu.skl_gemm_mxf4e2m1r_mxf4e2m1c_f32rc_gfx950(8, 8, 64, 1.0, a, lda, a, lsa, a, ldb, a, lsb, 0.0, c, 8, 1)
        assert gpu.skl_hip_last_error() == -2
    gpu.skl_gemm_mxf4e2m1r_mxf4e2m1c_f32rc_gfx950(8, 8, 64, 1.0, a, 64, None, 2, a, 64, a, 2, 0.0, c, 8, 1)
    assert gpu.skl_hip_last_error() == -2
    dev = DeviceBuffer.from_array(a)
    gpu.skl_gemm_mxf4e2m1r_mxf4e2m1c_f32rc_gfx950(8, 8, 64, 1.0, dev, 64, a, 2, a, 64, a, 2, 0.0, c, 8, 1)
    assert gpu.skl_hip_last_error() == -1
    assert (c == 3.0).all()


def test_a_training_step_against_differences(gpu):
    """dx and dW of L = sum(dy * y) through the quantisers as they are: with operands that MXFP4 holds exactly, the products are the
    derivatives of L, which is linear in x and in W, so differences give them back up to fp32's rounding of L itself."""
    rng = np.random.default_rng(12)
    m, n, k = 33, 70, 101
    x, w, dy = (rng.choice([-3.0, -1.0, 0.5, 2.0, 6.0], size=s).astype(np.float32) for s in ((m, k), (n, k), (m, n)))
    lib = gpu

    def quantised(v, across):
        rows, cols = (v.shape[1], v.shape[0]) if across else v.shape
        rs, cs = (1, v.shape[1]) if across else (v.shape[1], 1)
        ld, lds = cols + cols % 2, -(-cols // 32)
        src, dst, sc = DeviceBuffer.from_array(v), DeviceBuffer(rows * ld // 2), DeviceBuffer(rows * lds)
        lib.skl_cvt_f32rc_mxf4e2m1_gfx950(rows, cols, src, rs, cs, dst, ld, sc, lds)
        return rows, cols, dst, ld, sc, lds, src

    def product(a, b):
        out = DeviceBuffer(4 * a[0] * b[0])
        lib.skl_gemm_mxf4e2m1r_mxf4e2m1c_f32rc_gfx950(a[0], b[0], a[1], 1.0, a[2], a[3], a[4], a[5], b[2], b[3], b[4], b[5], 0.0, out, b[0], 1)
        _finish(lib)
        return out.download(np.float32).reshape(a[0], b[0]).astype(np.float64)

    y = product(quantised(x, False), quantised(w, False))
    dx = product(quantised(dy, False), quantised(w, True))
    dw = product(quantised(dy, True), quantised(x, True))
    x, w, dy = (v.astype(np.float64) for v in (x, w, dy))
    assert np.array_equal(y, x @ w.T) and np.array_equal(dx, dy @ w) and np.array_equal(dw, dy.T @ x)  # small whole multiples of a quarter
    loss = lambda x_, w_: float((dy * (x_ @ w_.T)).sum())  # noqa: E731
    for i, p in ((0, 0), (5, 99), (32, 100)):
        step = np.zeros_like(x)
        step[i, p] = 0.5
        assert loss(x + step, w) - loss(x - step, w) == dx[i, p]
        step = np.zeros_like(w)
        step[2 * i, p] = 0.5
        assert loss(x, w + step) - loss(x, w - step) == dw[2 * i, p]

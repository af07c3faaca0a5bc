"""Products grouped by expert where the values that rows meet are infinite: the same result whatever layout, alignment and kernel the operands have. All sums are of whole numbers
of few bits or not finite, so every result is exact."""
import numpy as np
import pytest

import grouped_support as gs
import skl_amd
from skl_amd import DeviceBuffer, U4Weights
from test_gpu_gemm_grouped import strided

pytestmark = pytest.mark.gpu

INF = {"bf16": 0x7F80, "f16": 0x7C00}


def download(lib, buf, *shape):
    assert lib.skl_hip_synchronize() == 0
    skl_amd.check_error()
    return buf.download(np.float32).reshape(shape)


# On 16-byte boundaries, where the streaming kernels run, and off them.
@pytest.mark.parametrize("pad", (8, 1))
@pytest.mark.parametrize("kind", ("bf16", "f16"))
def test_an_operand_without_rows(gpu, kind, pad):
    """An index into an A (or B) of no rows: nothing is multiplied, C = beta C, infinities in the other operand or not."""
    m, n, k = 70, 72, 64
    index, offsets = DeviceBuffer.from_array(np.zeros(m, np.int32)), DeviceBuffer.from_array(np.array([0, 30, 65], np.int32))
    other = DeviceBuffer.from_array(np.full((2 * n + m) * (n + pad), INF[kind], np.uint16))
    c = DeviceBuffer(4 * 2 * 72 * n)
    old = np.full(2 * 72 * n, 4.0, np.float32)
    grouped, over = (getattr(gpu, f"skl_gemm_grouped_{kind}_{kind}rc_f32_gfx950"), getattr(gpu, f"skl_gemm_groupedk_{kind}c_{kind}_f32_gfx950"))
    for strides in ((1, k + pad), (n + pad, 1)):
        c.upload(old)
        grouped(2, offsets, m, n, k, 1.0, None, k + pad, index, 0, other, *strides, n * (k + pad), 0.5, c, n)
        got = download(gpu, c, 2 * 72, n)
        assert np.all(got[:65] == 2.0) and np.all(got[65:] == 4.0), strides
    for rows in (("a",), ("b",), ("a", "b")):
        c.upload(old)
        a = (None, k + pad, index, 0) if "a" in rows else (other, k + pad, None, 0)
        b = (None, n + pad, index, 0) if "b" in rows else (other, n + pad, None, 0)
        over(2, offsets, k, n, m, 1.0, *a, *b, 0.5, c, n, 72 * n)
        got = download(gpu, c, 2, 72, n)
        assert np.all(got[:, :k] == 2.0) and np.all(got[:, k:] == 4.0), rows


@pytest.mark.parametrize("shift", (0, 1))
@pytest.mark.parametrize("m", (1, 3, 40))
def test_an_operand_without_rows_and_4_bit_weights(gpu, m, shift):
    n, k = 40, 64
    index = DeviceBuffer.from_array(np.zeros(m, np.int32))
    codes, scales = DeviceBuffer.from_array(np.full(n * k // 2 + 16, 0x33, np.uint8)), DeviceBuffer.from_array(np.full(n * 2, INF["bf16"], np.uint16))
    c = DeviceBuffer.from_array(np.full(m * n, 4.0, np.float32))
    w = U4Weights(group_k=32, codes=codes.offset(shift), ld=k, expert=0, scales=scales, zeros=None, ld_scales=2, expert_scales=0)
    gpu.skl_gemm_grouped_bf16_u4c_f32_gfx950(1, None, m, n, k, 1.0, None, k, index, 0, w, 0.5, c, n)
    assert np.all(download(gpu, c, m, n) == 2.0)


@pytest.mark.parametrize("pad", (8, 1))
@pytest.mark.parametrize("m", (2, 30, 300))
def test_a_row_outside_meets_infinite_weights(gpu, m, pad):
    """A row whose index is outside A is a row of zeros: NaN where a weight is infinite, 0 elsewhere."""
    n, k = 72, 64
    index, outside = np.arange(m) % 5, np.arange(1, m, 3)
    index[outside] = np.resize([-1, 5, 2 ** 31 - 1, -2 ** 31], len(outside))
    w = np.ones((n, k), np.float32)
    w[::4, 7] = np.inf
    a, b = strided(gs.bits(np.ones((5, k)), "bf16"), k + pad, 0), strided(gs.bits(w, "bf16"), k + pad, 0)
    da, db, di, c = DeviceBuffer.from_array(a), DeviceBuffer.from_array(b), DeviceBuffer.from_array(index.astype(np.int32)), DeviceBuffer(4 * m * n)
    gpu.skl_gemm_grouped_bf16_bf16rc_f32_gfx950(1, None, m, n, k, 1.0, da, k + pad, di, 5, db, 1, k + pad, 0, 0.0, c, n)
    got = download(gpu, c, m, n)
    want = np.full((m, n), 64.0)
    want[:, ::4], want[outside] = np.inf, 0.0
    want[outside, ::4] = np.nan
    assert np.array_equal(got, want, equal_nan=True)


@pytest.mark.parametrize("shift", (0, 1))
@pytest.mark.parametrize("kind", ("bf16", "f16"))
@pytest.mark.parametrize("k,group_k", [(64, 32), (192, 64), (256, 128), (96, 96)])
@pytest.mark.parametrize("m,n", [(1, 40), (2, 33), (30, 72), (300, 40)])
def test_a_row_outside_meets_infinite_scales(gpu, m, n, k, group_k, kind, shift):
    """With 4-bit weights, whose scales meet sums, such a row has none: 0, infinite scales or not - from the stream over the codes and, with codes off 16-byte boundaries, from the kernel
    for any layout."""
    blocks = -(-k // group_k)
    index, outside = np.arange(m) % 5, np.arange(min(1, m - 1), m, 3)
    index[outside] = np.resize([-1, 5, 2 ** 31 - 1, -2 ** 31], len(outside))
    scales = np.ones((n, blocks), np.float32)
    scales[::4, blocks // 2] = np.inf
    codes = np.concatenate([np.zeros(shift, np.uint8), gs.u4_store(np.full((n, k), 9, np.uint8), k)])
    da, di, dc, ds = (DeviceBuffer.from_array(v) for v in (gs.bits(np.ones((5, k)), kind), index.astype(np.int32), codes, gs.bits(scales, kind)))
    c = DeviceBuffer(4 * m * n)
    w = U4Weights(group_k=group_k, codes=dc.offset(shift), ld=k, expert=0, scales=ds, zeros=None, ld_scales=blocks, expert_scales=0)
    getattr(gpu, f"skl_gemm_grouped_{kind}_u4c_f32_gfx950")(1, None, m, n, k, 1.0, da, k, di, 5, w, 0.0, c, n)
    got = download(gpu, c, m, n)
    want = np.full((m, n), float(k))
    want[:, ::4], want[outside] = np.inf, 0.0
    assert np.array_equal(got, want)


@pytest.mark.parametrize("shift", (0, 1))
@pytest.mark.parametrize("kind", ("bf16", "f16"))
@pytest.mark.parametrize("k,group_k", [(128, 128), (64, 64), (384, 384), (100, 200), (512, 256)])
@pytest.mark.parametrize("m", (1, 3, 20))
def test_an_infinite_scale_meets_the_sum_of_128_values(gpu, m, k, group_k, kind, shift):
    """Every other 32 codes equal their zero point, so that their products are zeros: what an infinite scale meets is the sum of up to 128 values of the group, which is not."""
    n, blocks = 33, -(-k // group_k)
    q = np.full((n, k), 8, np.uint8)
    q[:, 32:64], q[:, 96:128] = 9, 11
    q[:, 128:] = 10
    q[1::2] = 16 - q[1::2]
    codes = np.concatenate([np.zeros(shift, np.uint8), gs.u4_store(q, k)])
    da, dc, ds = (DeviceBuffer.from_array(v) for v in (gs.bits(np.ones((m, k)), kind), codes, np.full((n, blocks), INF[kind], np.uint16)))
    c = DeviceBuffer(4 * m * n)
    w = U4Weights(group_k=group_k, codes=dc.offset(shift), ld=k, expert=0, scales=ds, zeros=None, ld_scales=blocks, expert_scales=0)
    getattr(gpu, f"skl_gemm_grouped_{kind}_u4c_f32_gfx950")(1, None, m, n, k, 1.0, da, k, None, 0, w, 0.0, c, n)
    got = download(gpu, c, m, n)
    assert np.all(got[:, 0::2] == np.inf) and np.all(got[:, 1::2] == -np.inf)

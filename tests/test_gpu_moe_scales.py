"""The mixture-of-experts layer at the ends of its weights' scales: 2^-127, the values that bf16 does not hold, and blocks that are no numbers."""
import numpy as np
import pytest

import mx_support as mx
import skl_amd
from gpu_support import _finish
from skl_amd import DeviceBuffer, MoeLayer

pytestmark = pytest.mark.gpu


def run(lib, x, codes, scales, hidden, inter):
    """y of one expert without activation, x (tokens, hidden); codes and scales by name."""
    t = x.shape[0]
    arrays = {}
    for name in ("gate", "up", "down"):
        flat = codes[name].reshape(-1)
        arrays[name] = DeviceBuffer.from_array(flat[0::2] | (flat[1::2] << 4))
        arrays[name + "_scales"] = DeviceBuffer.from_array(scales[name].reshape(-1))
    router, dx, y = DeviceBuffer.from_array(np.zeros(hidden, np.uint16)), DeviceBuffer.from_array(mx.to_bf16(x)), DeviceBuffer(4 * t * hidden)
    layer = MoeLayer(hidden=hidden, inter=inter, experts=1, top_k=1, router=router, ld_router=hidden, activation=0, normalise=1, ld_in=hidden, expert_in=0,
                     ld_in_scales=hidden // 32, expert_in_scales=0, ld_down=inter, expert_down=0, ld_down_scales=inter // 32, expert_down_scales=0, **arrays)
    lib.skl_moe_bf16_mxf4e2m1_f32_gfx950(layer, t, dx, hidden, 0.0, None, 0, y, hidden)
    _finish(lib)
    skl_amd.check_error()
    return y.download(np.float32).reshape(t, hidden)


def weights(rng, hidden, inter, low, high):
    shape = {"gate": (inter, hidden), "up": (inter, hidden), "down": (hidden, inter)}
    codes = {n: rng.integers(0, 16, size=s, dtype=np.uint8) for n, s in shape.items()}
    scales = {n: rng.integers(low, high, size=(s[0], s[1] // 32), dtype=np.uint8) for n, s in shape.items()}
    return codes, scales


@pytest.mark.parametrize("byte", (0, 1, 2))
@pytest.mark.parametrize("tokens,hidden,inter", ((1, 32, 32), (3, 320, 96), (20, 96, 288)))
def test_the_smallest_scales(gpu, byte, tokens, hidden, inter):
    """gate and up times 2^-127 and little more, x large: h of ordinary size. Whole numbers in every sum, so the bound is that of the terms of h."""
    rng = np.random.default_rng(byte + hidden)
    codes, scales = weights(rng, hidden, inter, 124, 128)
    scales["gate"][:], scales["up"][:] = byte, byte
    x = np.ldexp(rng.integers(-3, 4, size=(tokens, hidden)).astype(np.float64), 126 - 8)
    w = {n: mx.values(codes[n], scales[n]) for n in codes}
    h = (x @ w["gate"].T) * (x @ w["up"].T)
    want = h @ w["down"].T
    got = run(gpu, x.astype(np.float32), codes, scales, hidden, inter)
    bound = ((hidden + 2) * 4 + inter + 8 + 16) * mx.U * ((np.abs(x) @ np.abs(w["gate"]).T) * (np.abs(x) @ np.abs(w["up"]).T)) @ np.abs(w["down"]).T
    assert np.all(np.abs(got - want) <= bound), float((np.abs(got - want) / bound).max())
    assert np.abs(want).max() > 2.0 ** -30


def test_values_beyond_bf16_are_not_finite(gpu):
    """2^128 and more: 2, 3, 4 and 6 times 2^127, 4 and 6 times 2^126. An infinity, or NaN: one of the terms that its factor is held in can be zero."""
    hidden = inter = 32
    codes = {n: np.zeros((32, 32), np.uint8) for n in ("gate", "up", "down")}
    scales = {n: np.full((32, 1), 127, np.uint8) for n in codes}
    codes["gate"][0, 0] = codes["up"][0, 0] = 2                                  # h = (1, 0, ...)
    codes["down"][:16, 0] = codes["down"][16:, 0] = np.arange(16)
    scales["down"][:16], scales["down"][16:] = 254, 253
    x = np.zeros((1, 32), np.float32)
    x[0, 0] = 1.0
    got = run(gpu, x, codes, scales, hidden, inter)[0]
    magnitude = mx.MAGNITUDES[np.arange(8)]
    with np.errstate(over="ignore"):
        want = np.concatenate([np.concatenate([magnitude, -magnitude]) * s for s in (2.0 ** 127, 2.0 ** 126)]).astype(np.float32)
    assert np.isinf(want).sum() == 12
    assert np.array_equal(got[np.isfinite(want)], want[np.isfinite(want)]) and not np.isfinite(got[np.isinf(want)]).any()


def test_blocks_that_are_no_numbers(gpu):
    """In gate or up: that column of h, and with it every column of y of every token. In down: that column of y. In an expert that nobody chose: nothing."""
    rng = np.random.default_rng(3)
    hidden, inter = 288, 160
    x = rng.normal(size=(4, hidden)).astype(np.float32)
    codes, scales = weights(rng, hidden, inter, 120, 124)
    clean = run(gpu, x, codes, scales, hidden, inter)
    assert np.isfinite(clean).all()
    for name in ("gate", "up"):
        with_nan = {n: s.copy() for n, s in scales.items()}
        with_nan[name][70, 8] = 255
        assert np.isnan(run(gpu, x, codes, with_nan, hidden, inter)).all()
    with_nan = {n: s.copy() for n, s in scales.items()}
    with_nan["down"][100, 4] = 255
    got = run(gpu, x, codes, with_nan, hidden, inter)
    assert np.isnan(got[:, 100]).all()
    assert np.array_equal(np.delete(got, 100, axis=1), np.delete(clean, 100, axis=1))

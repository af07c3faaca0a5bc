"""A mixture-of-experts layer whose residual is its output: rows at the same distance are added to in place, others would be read where another token's have been
written and are refused - before anything is looked up, so that no GPU is needed to see it."""
import numpy as np
import pytest

import mx_support as mx
import skl_amd
from skl_amd import DeviceBuffer, MoeLayer

BAD_ARGUMENT = -2
HIDDEN, TOKENS = 32, 3


def layer(pointer=lambda v: v):
    codes, scales = np.zeros(2 * 32 * 16, np.uint8), np.full(2 * 32, 127, np.uint8)
    codes[:] = 0x22
    arrays = dict(router=np.zeros(2 * HIDDEN, np.uint16), gate=codes, up=codes, down=codes, gate_scales=scales, up_scales=scales, down_scales=scales)
    return MoeLayer(hidden=HIDDEN, inter=32, experts=2, top_k=1, ld_router=HIDDEN, ld_in=HIDDEN, expert_in=32 * HIDDEN, ld_in_scales=1, expert_in_scales=32,
                    ld_down=32, expert_down=32 * HIDDEN, ld_down_scales=1, expert_down_scales=32, activation=0, normalise=1, **{k: pointer(v) for k, v in arrays.items()})


def call(lib, layer_, x, tokens, beta, residual, ld_residual, y, ldy):
    lib.skl_hip_last_error()
    lib.skl_moe_bf16_mxf4e2m1_f32_gfx950(layer_, tokens, x, HIDDEN, beta, residual, ld_residual, y, ldy)
    return lib.skl_hip_last_error()


@pytest.mark.parametrize("ld_residual,ldy", ((32, 40), (40, 32), (64, 33)))
def test_other_distances_are_refused(ld_residual, ldy):
    lib = skl_amd.load()
    x, y = np.zeros((TOKENS, HIDDEN), np.uint16), np.full(TOKENS * 64, 3.0, np.float32)
    assert call(lib, layer(), x, TOKENS, 1.0, y, ld_residual, y, ldy) == BAD_ARGUMENT
    assert (y == 3.0).all()


@pytest.mark.gpu
def test_in_place_and_apart(gpu):
    x = mx.to_bf16(np.tile(np.arange(TOKENS, dtype=np.float32)[:, None], (1, HIDDEN)))
    start = np.arange(TOKENS * 64, dtype=np.float32)
    h = (np.arange(TOKENS) * 32.0) ** 2 * 32
    dev, dx = layer(DeviceBuffer.from_array), DeviceBuffer.from_array(x)
    for ld_residual, ldy, same, tokens, code in ((40, 40, True, 3, 0), (40, 48, True, 3, BAD_ARGUMENT), (40, 48, False, 3, 0), (7, 9, True, 1, 0)):
        y = DeviceBuffer.from_array(start)
        residual = y if same else DeviceBuffer.from_array(start)
        assert call(gpu, dev, dx, tokens, 1.0, residual, ld_residual, y, ldy) == code
        gpu.skl_hip_synchronize()
        want = start.copy()
        for t in range(tokens if code == 0 else 0):
            want[t * ldy:t * ldy + HIDDEN] = start[t * ld_residual:t * ld_residual + HIDDEN] + h[t]
        assert np.array_equal(y.download(np.float32), want), (ld_residual, ldy)
    # not read with beta == 0, so its distance does not count
    y = DeviceBuffer.from_array(start)
    assert call(gpu, dev, dx, 3, 0.0, y, 40, y, 48) == 0

"""The mixture-of-experts layer on the GPU against its definition in 64 bits, inside bounds derived from its fp32 sums (mx_support.moe)."""
import numpy as np
import pytest

import mx_support as mx
import skl_amd
from gpu_support import MODES, _finish
from skl_amd import DeviceBuffer, MoeLayer

pytestmark = pytest.mark.gpu


class Layer:
    """Random weights of a layer: as MXFP4 arrays with gaps of `pad` blocks between rows and experts, and as values."""

    def __init__(self, seed, hidden, inter, experts, pad=0):
        rng = self.rng = np.random.default_rng(seed)
        self.hidden, self.inter, self.experts = hidden, inter, experts
        self.router = mx.to_bf16((rng.normal(size=(experts, hidden + 8 * pad)) * 2 / np.sqrt(hidden)).astype(np.float32))
        self.members, self.value = {}, {}
        for name, rows, k in (("gate", inter, hidden), ("up", inter, hidden), ("down", hidden, inter)):
            ld, lds = k + 32 * pad, k // 32 + pad
            code = rng.integers(0, 16, size=(experts, rows, ld), dtype=np.uint8)
            scale = rng.integers(118, 125, size=(experts, rows, lds), dtype=np.uint8)
            group = "in" if name != "down" else "down"
            self.members[name] = code.reshape(-1)[0::2] | (code.reshape(-1)[1::2] << 4)
            self.members[name + "_scales"] = scale.reshape(-1).copy()
            self.members.update({f"ld_{group}": ld, f"expert_{group}": rows * ld, f"ld_{group}_scales": lds, f"expert_{group}_scales": rows * lds})
            self.value[name] = np.stack([mx.values(code[e][:, :k], scale[e][:, :k // 32]) for e in range(experts)])

    def run(self, lib, mode, x, top, act=2, normalise=True, beta=0.0, residual=None, want_choice=True, ldy=None):
        t = x.shape[0]
        ldy = self.hidden if ldy is None else ldy
        y, ids, weights = np.full(t * ldy, 5.0, np.float32), np.full(t * top, -1, np.int32), np.full(t * top, -1.0, np.float32)
        scalars = {k: v for k, v in self.members.items() if not isinstance(v, np.ndarray)}
        arrays = {k: v for k, v in self.members.items() if isinstance(v, np.ndarray)}
        arrays["router"] = self.router.reshape(-1)
        if want_choice:
            arrays.update(ids=ids, weights=weights)
        flat = np.ascontiguousarray(x)
        res = None if residual is None else np.ascontiguousarray(residual, np.float32)
        dev = {}
        if mode == "device":
            dev = {k: DeviceBuffer.from_array(v) for k, v in arrays.items()}
            flat, y_, res = DeviceBuffer.from_array(flat), DeviceBuffer.from_array(y), None if res is None else DeviceBuffer.from_array(res)
        else:
            y_ = y
        layer = MoeLayer(hidden=self.hidden, inter=self.inter, experts=self.experts, top_k=top, ld_router=self.router.shape[1], activation=act,
                         normalise=normalise, **scalars, **(dev or arrays))
        lib.skl_moe_bf16_mxf4e2m1_f32_gfx950(layer, t, flat, x.shape[1], beta, res, self.hidden, y_, ldy)
        if mode == "device":
            _finish(lib)
            y = y_.download(np.float32)
            if want_choice:
                ids, weights = dev["ids"].download(np.int32), dev["weights"].download(np.float32)
        skl_amd.check_error()
        return y.reshape(t, ldy), ids.reshape(t, top), weights.reshape(t, top)

    def check(self, lib, mode, tokens, top, act=2, normalise=True, beta=0.0, pad_x=0):
        x = mx.to_bf16(self.rng.normal(size=(tokens, self.hidden + 8 * pad_x)).astype(np.float32))
        residual = self.rng.normal(size=(tokens, self.hidden)).astype(np.float32) if beta else None
        xv = mx.of_bf16(x)[:, :self.hidden].astype(np.float64)
        got, got_ids, got_weights = self.run(lib, mode, x, top, act, normalise, beta, residual, ldy=self.hidden + 3)
        y, weights, bound, dw = mx.moe(xv, mx.of_bf16(self.router)[:, :self.hidden].astype(np.float64), self.value["gate"], self.value["up"],
                                       self.value["down"], top, act, normalise, beta, None if residual is None else residual.astype(np.float64), got_ids)
        assert np.all(np.abs(got_weights - weights) <= dw * weights), float((np.abs(got_weights - weights) / (dw * weights)).max())
        err = np.abs(got[:, :self.hidden] - y)
        assert np.all(err <= bound), float((err / bound).max())
        assert (got[:, self.hidden:] == 5.0).all(), "elements outside y were written"
        again, _, _ = self.run(lib, mode, x, top, act, normalise, beta, residual, want_choice=False, ldy=self.hidden + 3)
        assert np.array_equal(got.view(np.uint32), again.view(np.uint32)), "another result on the second run"


@pytest.mark.parametrize("hidden,inter,experts,top", ((32, 32, 1, 1), (64, 96, 4, 4), (160, 224, 5, 2), (512, 256, 16, 3), (1056, 544, 9, 2), (256, 2080, 3, 1),
                                                     (96, 64, 130, 8), (2048, 128, 70, 4)))
def test_layers(gpu, hidden, inter, experts, top):
    layer = Layer(hidden + inter, hidden, inter, experts)
    for mode, tokens, beta in (("device", 1, 0.0), ("device", 2, 1.0), ("host", 5, 0.5), ("device", 16, 0.0), ("device", 17, 1.0), ("device", 40, 0.0), ("device", 64, 1.0)):
        layer.check(gpu, mode, tokens, top, beta=beta)


@pytest.mark.parametrize("act", (0, 1, 2, 3))
@pytest.mark.parametrize("normalise", (False, True))
def test_activations_and_both_sums_of_the_softmax(gpu, act, normalise):
    Layer(act, 288, 160, 7, pad=1).check(gpu, "device", 9, 3, act=act, normalise=normalise, beta=1.0, pad_x=2)


def test_more_tokens_than_a_pass_takes(gpu):
    layer = Layer(77, 128, 96, 6)
    layer.check(gpu, "device", 65, 2, beta=1.0)
    layer.check(gpu, "host", 150, 3)


def test_all_tokens_choose_one_expert(gpu):
    """And most experts get none."""
    layer = Layer(5, 192, 128, 40)
    values = np.zeros((40, 192), np.float32)
    values[33] = 1.0
    layer.router = mx.to_bf16(values)
    x = mx.to_bf16(np.abs(layer.rng.normal(size=(50, 192)).astype(np.float32)) + 0.5)
    got, got_ids, got_weights = layer.run(gpu, "device", x, 1)
    y, _, bound, _ = mx.moe(mx.of_bf16(x).astype(np.float64), values.astype(np.float64), layer.value["gate"], layer.value["up"], layer.value["down"],
                            1, 2, True, 0.0, None, got_ids)
    assert (got_ids == 33).all() and (got_weights == 1.0).all()
    assert np.all(np.abs(got - y) <= bound)


def test_ties_go_to_the_lowest_expert(gpu):
    """Logits that are equal, whole numbers: the order is by logit and then by index; a zero's sign counts for nothing."""
    layer = Layer(6, 64, 32, 200)
    rng = layer.rng
    values = np.zeros((200, 64), np.float32)
    values[:, 0] = rng.integers(-2, 3, size=200)
    layer.router = mx.to_bf16(values)
    x = np.zeros((6, 64), np.float32)
    x[:, 0] = (1, -1, 2, 0, -0.0, 4)
    _, ids, weights = layer.run(gpu, "device", mx.to_bf16(x), 8)
    logits = x[:, :1].astype(np.float64) * values[:, 0][None, :]
    want = np.argsort(-(logits + 0.0), axis=1, kind="stable")[:, :8]
    assert np.array_equal(ids, want)
    picked = np.take_along_axis(logits, want, axis=1)
    exact = np.exp(picked - picked[:, :1])
    assert np.allclose(weights, exact / exact.sum(axis=1, keepdims=True), rtol=24 * mx.U * 8, atol=0)


def test_logits_that_are_not_numbers(gpu):
    """NaN logits are chosen last; a token of NaNs still names experts, the lowest, and makes NaN of its own row alone."""
    layer = Layer(7, 64, 32, 12)
    values = np.tile(np.arange(12, dtype=np.float32)[:, None], (1, 64)) / 64
    values[9:] = np.nan
    layer.router = (values.view(np.uint32) >> 16).astype(np.uint16)
    x = np.ones((3, 64), np.float32)
    x[1] = np.nan
    bits = (x.view(np.uint32) >> 16).astype(np.uint16)
    y, ids, weights = layer.run(gpu, "device", bits, 4)
    assert np.array_equal(ids[[0, 2]], [[8, 7, 6, 5]] * 2) and np.array_equal(ids[1], [0, 1, 2, 3])
    assert np.isfinite(weights[[0, 2]]).all() and np.isnan(weights[1]).all()
    assert np.isfinite(y[[0, 2]]).all() and np.isnan(y[1]).all()


def test_a_residual_in_place(gpu):
    layer = Layer(8, 96, 64, 4)
    x = mx.to_bf16(layer.rng.normal(size=(70, 96)).astype(np.float32))
    residual = layer.rng.normal(size=(70, 96)).astype(np.float32)
    apart, _, _ = layer.run(gpu, "device", x, 2, beta=0.75, residual=residual)
    arrays = {k: DeviceBuffer.from_array(v) for k, v in layer.members.items() if isinstance(v, np.ndarray)}
    scalars = {k: v for k, v in layer.members.items() if not isinstance(v, np.ndarray)}
    y, dx, router = DeviceBuffer.from_array(residual), DeviceBuffer.from_array(x), DeviceBuffer.from_array(layer.router)
    m = MoeLayer(hidden=96, inter=64, experts=4, top_k=2, router=router, ld_router=96, activation=2, normalise=1, **scalars, **arrays)
    gpu.skl_moe_bf16_mxf4e2m1_f32_gfx950(m, 70, dx, 96, 0.75, y, 96, y, 96)
    _finish(gpu)
    assert np.array_equal(y.download(np.float32).reshape(70, 96), apart)


def test_refusals(gpu):
    layer = Layer(9, 64, 32, 4)
    x, y = np.zeros((2, 64), np.uint16), np.full((2, 64), 3.0, np.float32)
    good = dict(hidden=64, inter=32, experts=4, top_k=2, router=layer.router.reshape(-1), ld_router=64, activation=2, normalise=1, **layer.members)

    def call(layer_=good, tokens=2, x_=x, ldx=64, beta=0.0, residual=None, ldy=64):
        gpu.skl_moe_bf16_mxf4e2m1_f32_gfx950(MoeLayer(**layer_) if layer_ else None, tokens, x_, ldx, beta, residual, 64, y, ldy)
        return gpu.skl_hip_last_error()

    bad = [dict(hidden=48), dict(inter=33), dict(hidden=0), dict(experts=0), dict(experts=1025), dict(top_k=0), dict(top_k=5), dict(activation=4), dict(activation=-1),
           dict(router=None), dict(gate=None), dict(down_scales=None), dict(ld_in=48), dict(ld_in=32), dict(ld_down=16), dict(expert_in=16), dict(ld_router=60),
           dict(ld_in_scales=1), dict(ld_down_scales=0)]
    for change in bad:
        assert call(dict(good, **change)) == -2, change
    assert call(None) == -2 and call(beta=1.0) == -2 and call(ldx=60) == -2 and call(ldy=63) == -2 and call(x_=None) == -2
    dev = DeviceBuffer.from_array(x)
    assert call(x_=dev) == -1
    assert call(tokens=0) == 0
    assert (y == 3.0).all()
    with pytest.raises(TypeError):
        MoeLayer(hiden=64)

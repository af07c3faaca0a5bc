"""examples/mxf4_layers.py: training on MXFP4 products takes the loss down, and the mixture-of-experts layer gives what its weights read back say; the gradients of a layer
of products of quantised operands against their formula and, for operands that quantise exactly, against differences."""
import importlib.util
import os

import numpy as np
import pytest

import mx_support as mx

pytestmark = pytest.mark.gpu

_PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "mxf4_layers.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("mxf4_layers", _PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_the_example_learns_and_answers(gpu, example):
    losses = example.train(gpu)
    assert np.isfinite(losses).all() and np.mean(losses[-5:]) < 0.5 * np.mean(losses[:3])
    # sums of 256 and 160 products on either side of an activation: far inside 2^-24 times the terms of a dot product of that length
    assert example.serve(gpu) < 1e-5


def test_gradients_against_the_formula(gpu, example):
    """dx = Q(dy) Q(W^T)^T and dW = Q(dy^T) Q(x^T)^T, each inside the bound of its sums."""
    rng = np.random.default_rng(5)
    layer = example.Linear(rng, 80, 96, 130)
    x, dy, w = rng.normal(size=(80, 96)).astype(np.float32), rng.normal(size=(80, 130)).astype(np.float32), layer.w.copy()
    y = layer.forward(gpu, x)
    dx = layer.backward(gpu, dy, 0.0)
    dw = layer.dw.download(np.float32).reshape(130, 96)
    q = lambda v: mx.values(*mx.quantise(v))
    for got, a, b in ((y, q(x), q(w)), (dx, q(dy), q(w.T)), (dw, q(dy.T), q(x.T))):
        want, bound = mx.product_bound(a, b, 1.0, 0.0, 0.0)
        assert np.all(np.abs(got - want) <= bound)


def test_gradients_against_differences(gpu, example):
    """Operands that MXFP4 holds exactly, along either axis: the quantisers are the identity there, and the derivative of sum(dy * y) is a difference of the
    layer's own outputs, exact in fp32: y is linear, and every number here a small multiple of 1/8."""
    rng = np.random.default_rng(6)
    layer = example.Linear(rng, 64, 32, 64)
    values = np.array([0.5, 1.0, 2.0, 4.0, 6.0])  # a block with a 6 has a scale of one; both axes get one
    draw = lambda m, n: (rng.choice(values, (m, n)) * rng.choice([-1.0, 1.0], (m, n))).astype(np.float32)

    def with_sixes(v):
        for i in range(v.shape[0]):
            for b in range(0, v.shape[1], 32):
                v[i, b + i % 32] = 6.0  # every row's block, and every column's, holds one
        return v

    x, w, dy = with_sixes(draw(64, 32)), with_sixes(draw(64, 32)), with_sixes(draw(64, 64))
    layer.w[:] = w
    layer.dev_w.upload(layer.w)
    loss = lambda: float((layer.forward(gpu, x).astype(np.float64) * dy).sum())
    base = loss()
    dx = layer.backward(gpu, dy, 0.0)
    dw = layer.dw.download(np.float32).reshape(64, 32)
    for i, p in ((0, 1), (5, 30), (63, 17)):  # not a 6, changed to another value of the grid
        old = x[i, p]
        x[i, p] = 0.5 if abs(old) != 0.5 else 1.0
        assert loss() - base == pytest.approx(float(dx[i, p]) * (x[i, p] - old), abs=0)
        x[i, p] = old
        old = layer.w[i, p]
        layer.w[i, p] = 0.5 if abs(old) != 0.5 else 1.0
        layer.dev_w.upload(layer.w)
        assert loss() - base == pytest.approx(float(dw[i, p]) * (layer.w[i, p] - old), abs=0)
        layer.w[i, p] = old
        layer.dev_w.upload(layer.w)

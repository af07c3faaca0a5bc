"""Layers with microscaled 4-bit (MXFP4) operands: two linear layers trained on them, and a mixture-of-experts layer that answers with them.

    python examples/mxf4_layers.py

Training: every product of a step - y = x W^T, dx = dy W, dW = dy^T x - multiplies MXFP4 operands, each quantised along the axis that its product
sums over; master weights, gradients and the update stay in fp32, and the gradients pass the quantisers as they are. Answering: an expert's weights
are quantised once, tokens come one by one or a few at a time. Needs the built library and a GPU; data are made up.
"""
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import skl_amd  # noqa: E402
from skl_amd import DeviceBuffer, MoeLayer  # noqa: E402


class Quantised:
    """An MXFP4 matrix of m rows of k values, made of an fp32 matrix on the device - or of its transpose."""

    def __init__(self, m, k):
        self.m, self.k, self.ld, self.lds = m, k, k + k % 2, -(-k // 32)
        self.codes, self.scales = DeviceBuffer(m * self.ld // 2), DeviceBuffer(m * self.lds)

    def take(self, lib, src, transposed=False):
        strides = (1, self.m) if transposed else (self.k, 1)
        lib.skl_cvt_f32rc_mxf4e2m1_gfx950(self.m, self.k, src, *strides, self.codes, self.ld, self.scales, self.lds)
        return self


def product(lib, a, b, c):
    """c = a b^T"""
    lib.skl_gemm_mxf4e2m1r_mxf4e2m1c_f32rc_gfx950(a.m, b.m, a.k, 1.0, a.codes, a.ld, a.scales, a.lds, b.codes, b.ld, b.scales, b.lds, 0.0, c, b.m, 1)
    return c


class Linear:
    """y = x W^T for `rows` rows of x at a time."""

    def __init__(self, rng, rows, inputs, outputs):
        self.w = (rng.normal(size=(outputs, inputs)) / np.sqrt(inputs)).astype(np.float32)
        self.rows, self.inputs, self.outputs = rows, inputs, outputs
        self.dev_w, self.x, self.dy = DeviceBuffer.from_array(self.w), DeviceBuffer(4 * rows * inputs), DeviceBuffer(4 * rows * outputs)
        self.y, self.dx, self.dw = DeviceBuffer(4 * rows * outputs), DeviceBuffer(4 * rows * inputs), DeviceBuffer(4 * outputs * inputs)
        self.xr, self.xc = Quantised(rows, inputs), Quantised(inputs, rows)
        self.wr, self.wc = Quantised(outputs, inputs), Quantised(inputs, outputs)
        self.dyr, self.dyc = Quantised(rows, outputs), Quantised(outputs, rows)

    def forward(self, lib, x):
        self.x.upload(x)
        product(lib, self.xr.take(lib, self.x), self.wr.take(lib, self.dev_w), self.y)
        return self._out(lib, self.y, self.rows, self.outputs)

    def backward(self, lib, dy, rate):
        self.dy.upload(dy)
        product(lib, self.dyr.take(lib, self.dy), self.wc.take(lib, self.dev_w, transposed=True), self.dx)
        product(lib, self.dyc.take(lib, self.dy, transposed=True), self.xc.take(lib, self.x, transposed=True), self.dw)
        dx = self._out(lib, self.dx, self.rows, self.inputs)
        self.w -= rate * self._out(lib, self.dw, self.outputs, self.inputs)
        self.dev_w.upload(self.w)
        return dx

    @staticmethod
    def _out(lib, buf, m, n):
        lib.skl_hip_synchronize()
        return buf.download(np.float32).reshape(m, n)


def train(lib, steps=40, rows=256, width=128, rate=0.02, seed=0):
    """Losses of a regression onto a fixed random network's outputs, one per step."""
    rng = np.random.default_rng(seed)
    first, second = Linear(rng, rows, width, 2 * width), Linear(rng, rows, 2 * width, 32)
    goal = [(rng.normal(size=s) / np.sqrt(s[1])).astype(np.float32) for s in ((2 * width, width), (32, 2 * width))]
    losses = []
    for _ in range(steps):
        x = rng.normal(size=(rows, width)).astype(np.float32)
        want = np.maximum(x @ goal[0].T, 0.0) @ goal[1].T
        hidden = first.forward(lib, x)
        error = second.forward(lib, np.maximum(hidden, 0.0)) - want
        losses.append(float((error ** 2).mean()))
        back = second.backward(lib, 2.0 * error / rows, rate)
        first.backward(lib, np.where(hidden > 0.0, back, 0.0).astype(np.float32), rate)
    return losses


class Experts:
    """A mixture-of-experts layer made of fp32 weights, quantised on the device."""

    def __init__(self, lib, rng, hidden=256, inter=160, experts=8, top_k=2, tokens=8):
        self.hidden, self.tokens, self.top_k = hidden, tokens, top_k
        router = (rng.normal(size=(experts, hidden)) / np.sqrt(hidden) * 4).astype(np.float32)
        self.router = ((router.view(np.uint32) + 0x8000) >> 16).astype(np.uint16)  # bf16
        members, self.weights = {}, {}
        for name, rows, k in (("gate", inter, hidden), ("up", inter, hidden), ("down", hidden, inter)):
            w = DeviceBuffer.from_array((rng.normal(size=(experts * rows, k)) / np.sqrt(k)).astype(np.float32))
            q, back = Quantised(experts * rows, k).take(lib, w), DeviceBuffer(4 * experts * rows * k)
            lib.skl_cvt_mxf4e2m1_f32rc_gfx950(experts * rows, k, q.codes, q.ld, q.scales, q.lds, back, k, 1)
            lib.skl_hip_synchronize()
            self.weights[name] = back.download(np.float32).reshape(experts, rows, k)  # what the layer multiplies by
            members[name], members[name + "_scales"] = q.codes, q.scales
        self.ids = DeviceBuffer(4 * tokens * top_k)
        self.x, self.residual, self.y = DeviceBuffer(2 * tokens * hidden), DeviceBuffer(4 * tokens * hidden), DeviceBuffer(4 * tokens * hidden)
        self.layer = MoeLayer(hidden=hidden, inter=inter, experts=experts, top_k=top_k, router=DeviceBuffer.from_array(self.router), ld_router=hidden,
                              ld_in=hidden, expert_in=inter * hidden, ld_in_scales=hidden // 32, expert_in_scales=inter * hidden // 32,
                              ld_down=inter, expert_down=inter * hidden, ld_down_scales=inter // 32, expert_down_scales=inter * hidden // 32,
                              activation=2, normalise=True, ids=self.ids, **members)

    def answer(self, lib, x, residual):
        """(residual + layer(x), chosen experts) for a few tokens, x in bf16 as uint16."""
        t = x.shape[0]
        self.x.upload(x), self.residual.upload(residual)
        lib.skl_moe_bf16_mxf4e2m1_f32_gfx950(self.layer, t, self.x, self.hidden, 1.0, self.residual, self.hidden, self.y, self.hidden)
        lib.skl_hip_synchronize()
        skl_amd.check_error()
        return self.y.download(np.float32, t * self.hidden).reshape(t, -1), self.ids.download(np.int32, t * self.top_k).reshape(t, -1)

    def plainly(self, x, residual):
        """The same in 64 bits, with the weights read back."""
        x = (x.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
        logits = x @ (self.router.astype(np.uint32) << 16).view(np.float32).astype(np.float64).T
        ids = np.argsort(-logits, axis=1, kind="stable")[:, :self.top_k]
        y = residual.astype(np.float64)
        for t in range(x.shape[0]):
            share = np.exp(logits[t, ids[t]] - logits[t, ids[t]].max())
            for e, w in zip(ids[t], share / share.sum()):
                gate, up = self.weights["gate"][e] @ x[t], self.weights["up"][e] @ x[t]
                y[t] += w * (self.weights["down"][e] @ (gate / (1.0 + np.exp(-gate)) * up))
        return y, ids


def serve(lib, seed=1):
    """Largest difference from the same layer in 64 bits, relative to the largest output, over a first pass of several tokens and single ones after it."""
    rng = np.random.default_rng(seed)
    layer = Experts(lib, rng)
    worst = 0.0
    for tokens in (layer.tokens, 1, 1, 1):
        x = rng.normal(size=(tokens, layer.hidden)).astype(np.float32)
        x = ((x.view(np.uint32) + 0x8000) >> 16).astype(np.uint16)
        residual = rng.normal(size=(tokens, layer.hidden)).astype(np.float32)
        y, ids = layer.answer(lib, x, residual)
        want, want_ids = layer.plainly(x, residual)
        assert np.array_equal(ids, want_ids)
        worst = max(worst, float(np.abs(y - want).max() / np.abs(want).max()))
    return worst


def main():
    lib = skl_amd.load()
    if lib.skl_hip_init(0) != 0:
        skl_amd.check_error()
    losses = train(lib)
    print(f"training with MXFP4 products: loss {losses[0]:.4f} -> {losses[-1]:.4f} in {len(losses)} steps")
    print(f"mixture of experts over MXFP4 weights: off by {serve(lib):.1e} of the largest output")


if __name__ == "__main__":
    main()

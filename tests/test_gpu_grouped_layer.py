"""A layer of experts made of the products grouped by expert, as a program would run it: picks put in the order of their experts, products up through the index of tokens, products down,
combined; backward the gradients of the input, of both weights and of the tokens. In 64 bits and by differences; with the padding of a batch, captured into a graph, on
streams of the caller's, and where a stream finds no scratch memory."""
import ctypes as ct

import numpy as np
import pytest

import grouped_support as gs
import skl_amd
import test_gpu_scratch_limits as limits
from skl_amd import DeviceBuffer, U4Weights

pytestmark = pytest.mark.gpu


def activation(h):
    return h * np.tanh(h)


def slope(h):
    return np.tanh(h) + h * (1 - np.tanh(h) ** 2)


def loss(x, up, down, ids, share, g):
    """<g, y> with y_t = sum_j share_tj down_e act(up_e x_t), e = ids_tj; 64 bits. An id outside the experts adds nothing."""
    total = 0.0
    for t in range(len(x)):
        for j in range(ids.shape[1]):
            e = ids[t, j]
            if 0 <= e < len(up):
                total += share[t, j] * (g[t] @ (down[e] @ activation(up[e] @ x[t])))
    return total


class Layer:
    """Device side: 16-bit operands, fp32 products. Rows of picks are padded to the largest possible number."""

    def __init__(self, kind, tokens, top_k, experts, hidden, inter, seed):
        self.kind, self.tokens, self.top, self.experts, self.hidden, self.inter, self.rng = kind, tokens, top_k, experts, hidden, inter, np.random.default_rng(seed)
        self.picks = tokens * top_k
        B, P, h, i = DeviceBuffer, self.picks, hidden, inter
        self.x, self.ids, self.up, self.down = B(2 * tokens * h), B(4 * P), B(2 * experts * i * h), B(2 * experts * h * i)
        self.offsets, self.order, self.rows, self.place = B(4 * (experts + 1)), B(4 * P), B(4 * P), B(4 * P)
        self.pre, self.act, self.out = B(4 * P * i), B(2 * P * i), B(4 * P * h)
        self.dout, self.dact, self.dpre, self.dx = B(2 * P * h), B(4 * P * i), B(2 * P * i), B(4 * P * h)
        self.dup, self.ddown = B(4 * experts * i * h), B(4 * experts * h * i)

    def weights(self, scale=0.3):
        r, e, i, h = self.rng, self.experts, self.inter, self.hidden
        self.h_up, self.h_down = gs.bits(r.normal(size=(e, i, h)) * scale, self.kind), gs.bits(r.normal(size=(e, h, i)) * scale, self.kind)
        self.up.upload(self.h_up), self.down.upload(self.h_down)

    def order_rows(self, lib):
        lib.skl_group_rows_gfx950(self.picks, self.ids, self.top, self.experts, self.offsets, self.order, self.rows, self.place)

    def go_up(self, lib):
        h, i = self.hidden, self.inter
        getattr(lib, f"skl_gemm_grouped_{self.kind}_{self.kind}rc_f32_gfx950")(self.experts, self.offsets, self.picks, i, h, 1.0, self.x, h, self.rows, self.tokens, self.up, 1, h, i * h, 0.0, self.pre, i)

    def go_down(self, lib):
        h, i = self.hidden, self.inter
        getattr(lib, f"skl_gemm_grouped_{self.kind}_{self.kind}rc_f32_gfx950")(self.experts, self.offsets, self.picks, h, i, 1.0, self.act, i, None, 0, self.down, 1, i, h * i, 0.0, self.out, h)

    def back_down(self, lib):  # d act = d out down, d down = d out^T act
        h, i, k = self.hidden, self.inter, self.kind
        getattr(lib, f"skl_gemm_grouped_{k}_{k}rc_f32_gfx950")(self.experts, self.offsets, self.picks, i, h, 1.0, self.dout, h, None, 0, self.down, i, 1, h * i, 0.0, self.dact, i)
        getattr(lib, f"skl_gemm_groupedk_{k}c_{k}_f32_gfx950")(self.experts, self.offsets, h, i, self.picks, 1.0, self.dout, h, None, 0, self.act, i, None, 0, 0.0, self.ddown, i, h * i)

    def back_up(self, lib):  # d x by pick, d up = d pre^T x
        h, i, k = self.hidden, self.inter, self.kind
        getattr(lib, f"skl_gemm_grouped_{k}_{k}rc_f32_gfx950")(self.experts, self.offsets, self.picks, h, i, 1.0, self.dpre, i, None, 0, self.up, h, 1, i * h, 0.0, self.dx, h)
        getattr(lib, f"skl_gemm_groupedk_{k}c_{k}_f32_gfx950")(self.experts, self.offsets, i, h, self.picks, 1.0, self.dpre, i, None, 0, self.x, h, self.rows, self.tokens, 0.0, self.dup, h, i * h)


def picks_of(rng, tokens, top_k, experts, padded):
    ids = np.stack([rng.permutation(experts)[:top_k] for _ in range(tokens)]).astype(np.int32)
    ids[ids == experts - 1] = 0  # an expert without a token, a token that has one twice
    ids[tokens - padded:] = -1   # the padding of a batch
    return ids


@pytest.mark.parametrize("kind,tokens,hidden,inter", (("bf16", 37, 64, 96), ("f16", 150, 72, 40), ("bf16", 20, 31, 17)))
def test_a_layer_and_its_gradients(gpu, kind, tokens, hidden, inter):
    top, experts, padded = 3, 6, 5
    L = Layer(kind, tokens, top, experts, hidden, inter, hidden)
    rng = L.rng
    L.weights()
    ids, share = picks_of(rng, tokens, top, experts, padded), rng.uniform(0.1, 1, (tokens, top))
    hx, hg = gs.bits(rng.normal(size=(tokens, hidden)), kind), rng.normal(size=(tokens, hidden))
    L.x.upload(hx), L.ids.upload(ids)
    for buf in (L.order, L.rows, L.pre, L.out, L.dact, L.dx, L.dup, L.ddown, L.dout, L.act, L.dpre):
        gpu.skl_hip_memset(buf, 0xFF, buf.nbytes)  # NaN, -1
    L.order_rows(gpu)
    off, order, rows, place = gs.group_rows(ids.ravel(), top, experts)
    n = int(off[-1])
    assert n == top * (tokens - padded)
    got_offsets, got_order, got_rows, got_place = (b.download(np.int32) for b in (L.offsets, L.order, L.rows, L.place))
    assert np.array_equal(got_offsets, off) and np.array_equal(got_order[:n], order) and np.array_equal(got_rows[:n], rows) and np.array_equal(got_place, place)
    assert np.all(got_order[n:] == -1) and np.all(got_rows[n:] == -1)
    ranges = gs.cut(off, L.picks, experts)
    x, up, down = gs.values(hx, kind), gs.values(L.h_up, kind), gs.values(L.h_down, kind)

    def checked(buf, cols, want, bound, inside):
        got = buf.download(np.float32).reshape(L.picks, cols)
        assert np.isnan(got[~inside]).all() and np.all(np.abs(got[inside] - want[inside]) <= bound[inside])
        return got[:n].astype(np.float64)

    nothing = lambda cols: np.zeros((L.picks, cols))  # noqa: E731
    L.go_up(gpu)
    pre = checked(L.pre, inter, *gs.product(x, [w.T for w in up], nothing(inter), 1.0, 0.0, ranges, np.append(rows, np.full(L.picks - n, -1))))
    h_act = gs.bits(activation(pre), kind)
    L.act.upload(h_act)
    act = gs.values(h_act, kind)
    whole = lambda v: np.concatenate([v, np.zeros((L.picks - n, v.shape[1]))])  # noqa: E731
    L.go_down(gpu)
    out = checked(L.out, hidden, *gs.product(whole(act), [w.T for w in down], nothing(hidden), 1.0, 0.0, ranges))
    y = np.zeros((tokens, hidden))
    for p in range(n):
        y[rows[p]] += share.ravel()[order[p]] * out[p]
    assert np.all(y[tokens - padded:] == 0)
    # backward
    h_dout = gs.bits(share.ravel()[order][:, None] * hg[rows], kind)
    L.dout.upload(h_dout)
    dout = gs.values(h_dout, kind)
    L.back_down(gpu)
    dact = checked(L.dact, inter, *gs.product(whole(dout), list(down), nothing(inter), 1.0, 0.0, ranges))
    want, bound = gs.over(whole(dout), whole(act), np.zeros((experts, hidden, inter)), 1.0, 0.0, ranges, total=L.picks)
    ddown = L.ddown.download(np.float32).reshape(want.shape)
    assert np.all(np.abs(ddown - want) <= bound) and np.all(ddown[experts - 1] == 0)
    h_dpre = gs.bits(dact * slope(pre), kind)
    L.dpre.upload(h_dpre)
    dpre = gs.values(h_dpre, kind)
    L.back_up(gpu)
    by_pick = checked(L.dx, hidden, *gs.product(whole(dpre), list(up), nothing(hidden), 1.0, 0.0, ranges))
    want, bound = gs.over(whole(dpre), x, np.zeros((experts, inter, hidden)), 1.0, 0.0, ranges, None, np.append(rows, np.full(L.picks - n, -1)), total=L.picks)
    dup = L.dup.download(np.float32).reshape(want.shape)
    skl_amd.check_error()
    assert np.all(np.abs(dup - want) <= bound) and np.all(dup[experts - 1] == 0)
    dx = np.zeros((tokens, hidden))
    np.add.at(dx, rows, by_pick)
    # The gradients against differences of the loss along random directions. Two roundings are on the way of each: of the output's gradient, and of activations (down) or their
    # gradients (up, x), each at most half a step relative to a value, so both together at most two half steps of the same sums taken of magnitudes. As much again is left for the fp32 sums, whose
    # bounds of 75 * 2^-23 of magnitudes are fifty times smaller than half a step of f16, before and behind the activation, whose slope changes no faster than twice the value it is of. The
    # differences' own error: the square of a step of 1e-4 times the values it is multiplied with, 1e-5 at most.
    half = 2.0 ** -8 if kind == "bf16" else 2.0 ** -11
    for which, gradient, at in (("x", dx, x), ("up", dup, up), ("down", ddown, down)):
        for _ in range(2):
            v = rng.choice([-1.0, 1.0], at.shape)
            step = 1e-4

            def moved(s):
                here = dict(x=x, up=up, down=down)
                here[which] = at + s * step * v
                return loss(here["x"], here["up"], here["down"], ids, share, hg)
            slope_seen = (moved(1) - moved(-1)) / (2 * step)
            magnitudes = derivative_of_magnitudes(x, up, down, ids, share, hg, which)
            assert abs(slope_seen - np.sum(gradient.astype(np.float64) * v)) <= 4 * half * magnitudes, which


def derivative_of_magnitudes(x, up, down, ids, share, g, which):
    """The sum over `which` of the derivatives' sums of magnitudes: what roundings along the way are relative to."""
    total = 0.0
    for t in range(len(x)):
        for j in range(ids.shape[1]):
            e = ids[t, j]
            if not 0 <= e < len(up):
                continue
            dout = share[t, j] * np.abs(g[t])
            pre = up[e] @ x[t]
            if which == "down":
                total += dout.sum() * np.abs(activation(pre)).sum()
                continue
            dpre = (dout @ np.abs(down[e])) * np.abs(slope(pre))
            total += dpre.sum() * np.abs(x[t]).sum() if which == "up" else (dpre @ np.abs(up[e])).sum()
    return total


class Pass:
    """One run over everything that only enqueues: enough picks for the order's two launches, tiles of two sizes, 4-bit weights for one row and for many, an odd layout."""

    def __init__(self, seed):
        self.layer = L = Layer("bf16", 24000, 4, 16, 64, 96, seed)
        L.weights()
        rng = L.rng
        B, at = DeviceBuffer, DeviceBuffer.from_array
        L.act.upload(gs.bits(rng.normal(size=(L.picks, L.inter)), "bf16")), L.dout.upload(gs.bits(rng.normal(size=(L.picks, L.hidden)), "bf16"))
        L.dpre.upload(gs.bits(rng.normal(size=(L.picks, L.inter)), "bf16"))
        self.n, self.k = 1000, 1024
        self.codes, self.scales = at(rng.integers(0, 256, 3 * self.n * self.k // 2, dtype=np.uint8)), at(gs.bits(rng.uniform(0.01, 0.1, 3 * self.n * self.k // 128), "bf16"))
        self.zeros = at(rng.integers(0, 16, 3 * self.n * self.k // 128, dtype=np.uint8))
        self.tokens, self.parts = B(2 * 40 * self.k), at(np.array([0, 2, 30, 40], np.int32))
        self.one, self.many, self.odd = B(4 * self.n), B(4 * 40 * self.n), B(4 * L.picks * 31)
        self.outputs = dict(offsets=L.offsets, order=L.order, rows=L.rows, place=L.place, pre=L.pre, out=L.out, dact=L.dact, dx=L.dx, dup=L.dup, ddown=L.ddown, one=self.one, many=self.many, odd=self.odd)

    def next_input(self):
        L, rng = self.layer, self.layer.rng
        ids = rng.integers(-1, L.experts, L.picks).astype(np.int32)
        ids[rng.random(L.picks) < 0.3] = rng.integers(0, L.experts)
        L.ids.upload(ids), L.x.upload(gs.bits(rng.normal(size=(L.tokens, L.hidden)), "bf16")), self.tokens.upload(gs.bits(rng.normal(size=(40, self.k)), "bf16"))

    def enqueue(self, lib):
        L, n, k = self.layer, self.n, self.k
        L.order_rows(lib), L.go_up(lib), L.go_down(lib), L.back_down(lib), L.back_up(lib)
        w = U4Weights(group_k=128, codes=self.codes, ld=k, expert=n * k, scales=self.scales, zeros=self.zeros, ld_scales=k // 128, expert_scales=n * k // 128)
        lib.skl_gemm_grouped_bf16_u4c_f32_gfx950(1, None, 1, n, k, 1.0, self.tokens, k, None, 0, w, 0.0, self.one, n)
        lib.skl_gemm_grouped_bf16_u4c_f32_gfx950(3, self.parts, 40, n, k, 1.0, self.tokens, k, None, 0, w, 0.0, self.many, n)
        lib.skl_gemm_grouped_bf16_bf16rc_f32_gfx950(L.experts, L.offsets, L.picks, 31, 63, 1.0, L.x, L.hidden, L.rows, L.tokens, L.up, 1, 63, 31 * 63, 0.0, self.odd, 31)

    def spoil(self, lib):
        for buf in self.outputs.values():
            lib.skl_hip_memset(buf, 0x5A, buf.nbytes)

    def take(self, lib):
        assert lib.skl_hip_synchronize() == 0
        return {name: buf.download(np.uint8, buf.nbytes) for name, buf in self.outputs.items()}


@pytest.fixture()
def hip():
    lib = ct.CDLL("libamdhip64.so.7")
    for name in ("hipStreamCreate", "hipStreamBeginCapture", "hipStreamEndCapture", "hipGraphInstantiate", "hipGraphLaunch", "hipStreamSynchronize", "hipGraphExecDestroy",
                 "hipGraphDestroy", "hipStreamDestroy"):
        getattr(lib, name).restype = ct.c_int
    return lib


def same(got, want):
    for name in want:
        assert np.array_equal(got[name], want[name]), name


def test_replays_from_a_graph_give_the_eager_results(gpu, hip):
    work = Pass(1)
    stream, graph, executable = ct.c_void_p(), ct.c_void_p(), ct.c_void_p()
    assert hip.hipStreamCreate(ct.byref(stream)) == 0
    gpu.skl_hip_set_pointer_mode(1)
    gpu.skl_hip_set_stream(stream.value)
    try:
        work.next_input()
        work.spoil(gpu)
        work.enqueue(gpu)  # creates the stream's scratch memory and configures the kernels
        assert gpu.skl_hip_synchronize() == 0
        skl_amd.check_error()
        assert hip.hipStreamBeginCapture(stream, 0) == 0
        work.enqueue(gpu)
        assert hip.hipStreamEndCapture(stream, ct.byref(graph)) == 0
        skl_amd.check_error()
        assert hip.hipGraphInstantiate(ct.byref(executable), graph, None, None, ct.c_size_t(0)) == 0
        for _ in range(4):
            work.next_input()
            work.spoil(gpu)
            work.enqueue(gpu)
            want = work.take(gpu)
            work.spoil(gpu)
            assert gpu.skl_hip_synchronize() == 0
            assert hip.hipGraphLaunch(executable, stream) == 0
            assert hip.hipStreamSynchronize(stream) == 0
            same(work.take(gpu), want)
        skl_amd.check_error()
    finally:
        gpu.skl_hip_set_stream(None)
        gpu.skl_hip_set_pointer_mode(0)
        if executable:
            hip.hipGraphExecDestroy(executable)
        if graph:
            hip.hipGraphDestroy(graph)
        gpu.skl_hip_release_stream(stream.value)
        hip.hipStreamDestroy(stream)


def test_two_streams_at_once(gpu, hip):
    """Passes under way together, each with its own scratch memory, give what each gives alone."""
    work = [Pass(2), Pass(3)]
    streams = [ct.c_void_p(), ct.c_void_p()]
    gpu.skl_hip_set_pointer_mode(1)
    try:
        want = []
        for w in work:
            w.next_input()
            w.spoil(gpu)
            w.enqueue(gpu)
            want.append(w.take(gpu))
            w.spoil(gpu)
            assert gpu.skl_hip_synchronize() == 0
        for stream in streams:
            assert hip.hipStreamCreate(ct.byref(stream)) == 0
        for _ in range(3):
            for w, stream in zip(work, streams):
                gpu.skl_hip_set_stream(stream.value)
                w.enqueue(gpu)
        for w, stream, wanted in zip(work, streams, want):
            gpu.skl_hip_set_stream(stream.value)
            same(w.take(gpu), wanted)
        skl_amd.check_error()
    finally:
        gpu.skl_hip_set_stream(None)
        gpu.skl_hip_set_pointer_mode(0)
        for stream in streams:
            gpu.skl_hip_release_stream(stream.value)
            hip.hipStreamDestroy(stream)


def test_without_a_scratch_slot(gpu, hip):
    """A stream beyond those that hold scratch memory: the order comes from one workgroup, and is the same; gradients of few weights are summed in one part, which is another order."""
    work = Pass(4)
    gpu.skl_hip_set_pointer_mode(1)
    streams = []
    try:
        work.next_input()
        work.spoil(gpu)
        work.enqueue(gpu)
        want = work.take(gpu)
        skl_amd.check_error()
        streams = limits._streams_until_the_slots_are_gone(gpu, hip, ct)
        work.spoil(gpu)
        work.enqueue(gpu)
        got = work.take(gpu)
        assert gpu.skl_hip_last_error() == 0
        L = work.layer
        n, rows = int(want["offsets"].view(np.int32)[-1]), want["rows"].view(np.int32)
        ranges = gs.cut(want["offsets"].view(np.int32), L.picks, L.experts)
        load = lambda buf, cols: gs.values(buf.download(np.uint16).reshape(-1, cols), "bf16")  # noqa: E731
        index = np.append(rows[:n], np.full(L.picks - n, -1))
        sums = {"dup": gs.over(load(L.dpre, L.inter), load(L.x, L.hidden), np.zeros((L.experts, L.inter, L.hidden)), 1.0, 0.0, ranges, None, index, total=L.picks),
                "ddown": gs.over(load(L.dout, L.hidden), load(L.act, L.inter), np.zeros((L.experts, L.hidden, L.inter)), 1.0, 0.0, ranges, total=L.picks)}
        for name, (exact, bound) in sums.items():
            for side in (got, want):
                assert np.all(np.abs(side.pop(name).view(np.float32).reshape(exact.shape) - exact) <= bound), name
        same(got, want)
    finally:
        gpu.skl_hip_set_stream(None)
        gpu.skl_hip_set_pointer_mode(0)
        for stream in streams:
            gpu.skl_hip_release_stream(stream.value)
            hip.hipStreamDestroy(stream)
        gpu.skl_hip_last_error()


def test_beta_zero_as_the_reference_has_it(gpu):
    """With the reference's evaluation C is read and multiplied by zero: NaN stays NaN, everywhere that a group has rows."""
    rng = np.random.default_rng(6)
    a, w = gs.bits(rng.normal(size=(20, 64)), "bf16"), gs.bits(rng.normal(size=(2, 48, 64)), "bf16")
    da, dw, o = DeviceBuffer.from_array(a), DeviceBuffer.from_array(w), DeviceBuffer.from_array(np.array([0, 12, 18], np.int32))
    u4 = U4Weights(group_k=64, codes=dw, ld=64, expert=48 * 64, scales=da, zeros=None, ld_scales=1, expert_scales=48)
    c = DeviceBuffer(4 * 2 * 64 * 64)

    def calls():
        yield 18 * 48, lambda: gpu.skl_gemm_grouped_bf16_bf16rc_f32_gfx950(2, o, 20, 48, 64, 1.0, da, 64, None, 0, dw, 1, 64, 48 * 64, 0.0, c, 48)
        yield 18 * 48, lambda: gpu.skl_gemm_grouped_bf16_u4c_f32_gfx950(2, o, 20, 48, 64, 1.0, da, 64, None, 0, u4, 0.0, c, 48)
        yield 2 * 64 * 64, lambda: gpu.skl_gemm_groupedk_bf16c_bf16_f32_gfx950(2, o, 64, 64, 18, 1.0, da, 64, None, 0, da, 64, None, 0, 0.0, c, 64, 64 * 64)
    try:
        for mode, spoiled in ((1, True), (0, False)):
            gpu.skl_hip_set_beta_zero_mode(mode)
            for count, call in calls():
                gpu.skl_hip_memset(c, 0xFF, c.nbytes)
                call()
                got = c.download(np.float32)[:count]
                skl_amd.check_error()
                assert np.isnan(got).all() if spoiled else np.isfinite(got).all()
    finally:
        gpu.skl_hip_set_beta_zero_mode(0)

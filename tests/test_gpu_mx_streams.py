"""The microscaled 4-bit operators and the mixture-of-experts layer where a program's streams come in: captured into a graph and replayed, on a
stream of the caller's, and on one that finds no scratch memory left."""
import ctypes as ct

import numpy as np
import pytest

import mx_support as mx
import skl_amd
import test_gpu_scratch_limits as limits
from skl_amd import DeviceBuffer, MoeLayer

pytestmark = pytest.mark.gpu


class Pass:
    """Buffers of one pass: x (m, k) is quantised by rows and by columns and read back; two products, one of large tiles with rows off line
    boundaries and one whose small tiles share K; a mixture-of-experts layer on the first rows of x."""

    m, n, k, tokens, inter, experts, top = 2080, 2048, 1056, 40, 96, 12, 3

    def __init__(self, seed):
        m, n, k = self.m, self.n, self.k
        rng = np.random.default_rng(seed)
        B, at = DeviceBuffer, DeviceBuffer.from_array
        self.x = B(2 * m * k)
        self.w, self.ws = at(rng.integers(0, 256, n * k // 2, dtype=np.uint8)), at(rng.integers(120, 130, n * (k // 32), dtype=np.uint8))
        self.q, self.s, self.qt, self.st = B(m * k // 2), B(m * (k // 32)), B(k * m // 2), B(k * (m // 32))
        self.back, self.large, self.small = B(2 * m * k), B(4 * m * n), B(4 * 96 * 96)
        layer = {}
        for name, rows, cols in (("gate", self.inter, k), ("up", self.inter, k), ("down", k, self.inter)):
            layer[name] = at(rng.integers(0, 256, self.experts * rows * cols // 2, dtype=np.uint8))
            layer[name + "_scales"] = at(rng.integers(118, 124, self.experts * rows * cols // 32, dtype=np.uint8))
        layer["router"] = at(mx.to_bf16((rng.normal(size=self.experts * k) * 0.1).astype(np.float32)))
        self.y, self.ids = B(4 * self.tokens * k), B(4 * self.tokens * self.top)
        self.layer = MoeLayer(hidden=k, inter=self.inter, experts=self.experts, top_k=self.top, ld_router=k, activation=2, normalise=1, ids=self.ids,
                              ld_in=k, expert_in=self.inter * k, ld_in_scales=k // 32, expert_in_scales=self.inter * k // 32,
                              ld_down=self.inter, expert_down=self.inter * k, ld_down_scales=self.inter // 32, expert_down_scales=self.inter * k // 32, **layer)
        self.outputs = {"q": self.q, "s": self.s, "qt": self.qt, "st": self.st, "back": self.back, "large": self.large, "small": self.small, "y": self.y, "ids": self.ids}
        self.next_input = lambda: mx.to_bf16(rng.normal(size=m * k).astype(np.float32))

    def enqueue(self, lib):
        m, n, k = self.m, self.n, self.k
        lib.skl_cvt_bf16rc_mxf4e2m1_gfx950(m, k, self.x, k, 1, self.q, k, self.s, k // 32)
        lib.skl_cvt_bf16rc_mxf4e2m1_gfx950(k, m, self.x, 1, k, self.qt, m, self.st, m // 32)
        lib.skl_cvt_mxf4e2m1_bf16rc_gfx950(m, k, self.q, k, self.s, k // 32, self.back, k, 1)
        lib.skl_gemm_mxf4e2m1r_mxf4e2m1c_f32rc_gfx950(m, n, k, 1.0, self.q, k, self.s, k // 32, self.w, k, self.ws, k // 32, 0.0, self.large, n, 1)
        lib.skl_gemm_mxf4e2m1r_mxf4e2m1c_f32rc_gfx950(96, 96, m, 1.0, self.qt, m, self.st, m // 32, self.qt, m, self.st, m // 32, 0.0, self.small, 96, 1)
        lib.skl_moe_bf16_mxf4e2m1_f32_gfx950(self.layer, self.tokens, self.x, k, 0.0, None, 0, self.y, k)

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
        work.x.upload(work.next_input())
        work.enqueue(gpu)  # creates the stream's scratch memory and configures the kernels
        assert gpu.skl_hip_synchronize() == 0
        skl_amd.check_error()
        assert hip.hipStreamBeginCapture(stream, 0) == 0
        work.enqueue(gpu)
        assert hip.hipStreamEndCapture(stream, ct.byref(graph)) == 0
        skl_amd.check_error()
        assert hip.hipGraphInstantiate(ct.byref(executable), graph, None, None, ct.c_size_t(0)) == 0
        for _ in range(4):
            work.x.upload(work.next_input())
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
            w.x.upload(w.next_input())
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
    """A stream beyond those that hold scratch memory: products of large tiles read their operands as they lie, K is not shared, the layer takes a block of its own."""
    work = Pass(4)
    gpu.skl_hip_set_pointer_mode(1)
    streams = []
    try:
        work.x.upload(work.next_input())
        work.enqueue(gpu)
        want = work.take(gpu)
        skl_amd.check_error()
        streams = limits._streams_until_the_slots_are_gone(gpu, hip, ct)
        work.spoil(gpu)
        work.enqueue(gpu)
        got = work.take(gpu)
        assert gpu.skl_hip_last_error() == 0
        for name in ("large", "small"):  # fp32 sums in another order
            a, b = got.pop(name).view(np.float32).astype(np.float64), want.pop(name).view(np.float32).astype(np.float64)
            code, scales = mx.loaded(want["q"], want["s"], work.m, work.k, work.k, work.k // 32)
            if name == "large":
                w = work.w.download(np.uint8, work.w.nbytes), work.ws.download(np.uint8, work.ws.nbytes)
                other = mx.values(*mx.loaded(*w, work.n, work.k, work.k, work.k // 32))
                exact, bound = mx.product_bound(mx.values(code, scales), other, 1.0, 0.0, 0.0)
            else:
                t = mx.values(*mx.loaded(want["qt"], want["st"], work.k, work.m, work.m, work.m // 32))[:96]
                exact, bound = mx.product_bound(t, t, 1.0, 0.0, 0.0)
            assert np.all(np.abs(a.reshape(exact.shape) - exact) <= bound) and np.all(np.abs(b.reshape(exact.shape) - exact) <= bound)
        same(got, want)
    finally:
        gpu.skl_hip_set_stream(None)
        gpu.skl_hip_set_pointer_mode(0)
        for stream in streams:
            gpu.skl_hip_release_stream(stream.value)
            hip.hipStreamDestroy(stream)
        gpu.skl_hip_last_error()

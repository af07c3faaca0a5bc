"""Sums over groups of rows into matrices whose rows lie side by side: C_e(i, j) at c[e * gsc + i * rsc + j] with gsc less than a matrix, as [m][groups][n] has it."""
import os
import subprocess

import numpy as np
import pytest

import grouped_support as gs
import skl_amd
from skl_amd import DeviceBuffer

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_host_layer_takes_what_lies_apart(tmp_path):
    program = tmp_path / "host_layer_interleaved_check"
    clang = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "lib", "llvm", "bin", "clang")
    sources = [os.path.join(ROOT, *at) for at in (("skl_amd", "csrc", "skl_api_grouped.c"), ("tests", "c", "host_layer_interleaved_check.c"))]
    subprocess.run([clang, "-std=c11", "-O1", "-g", "-Wall", "-Wextra", "-Werror", "-fsanitize=address,undefined", "-fno-sanitize-recover=undefined", *sources, "-o", program], check=True)
    run = subprocess.run([program], capture_output=True, text=True, env=dict(os.environ, ASAN_OPTIONS="detect_leaks=0"))
    assert run.returncode == 0 and run.stdout == "interleaved ok\n", run.stdout + run.stderr


# Sums on the streaming kernel in one part and in several, and on the kernel for any layout.
@pytest.mark.gpu
@pytest.mark.parametrize("mode", ("device", "host"))
@pytest.mark.parametrize("m,n,lengths,pitch", ((72, 264, (70, 0, 33, 200), 8), (136, 128, (3000, 700), 8), (40, 33, (20, 1, 9), 1)))
def test_results_side_by_side(gpu, m, n, lengths, pitch, mode):
    groups, total = len(lengths), sum(lengths)
    rng = np.random.default_rng(m + n)
    a, b = (gs.bits(rng.integers(-4, 5, (total, cols)), "bf16") for cols in (m, n))  # sums of whole numbers: exact
    pa, pb = -m % pitch + m, -n % pitch + n
    fa, fb = np.zeros((total, pa), np.uint16), np.zeros((total, pb), np.uint16)
    fa[:, :m], fb[:, :n] = a, b
    offsets = np.concatenate(([0], np.cumsum(lengths))).astype(np.int32)
    gsc = n + 3
    rsc = groups * gsc + 1
    c = np.full(m * rsc, 4.0, np.float32)
    want = c.reshape(m, rsc).copy()
    for e in range(groups):
        x, y = (gs.values(v[offsets[e]:offsets[e + 1]], "bf16") for v in (a, b))
        want[:, e * gsc:e * gsc + n] = x.T @ y + 2.0
    args = lambda o, x, y, z: (groups, o, m, n, total, 1.0, x, pa, None, 0, y, pb, None, 0, 0.5, z, rsc, gsc)  # noqa: E731
    if mode == "host":
        got = c[:(groups - 1) * gsc + (m - 1) * rsc + n].copy()
        gpu.skl_gemm_groupedk_bf16c_bf16_f32_gfx950(*args(offsets, fa, fb, got))
        got = np.concatenate([got, c[len(got):]])
    else:
        bufs = [DeviceBuffer.from_array(v) for v in (offsets, fa, fb, c)]
        gpu.skl_gemm_groupedk_bf16c_bf16_f32_gfx950(*args(*bufs))
        got = bufs[3].download(np.float32)
    skl_amd.check_error()
    assert np.array_equal(got.reshape(m, rsc), want)

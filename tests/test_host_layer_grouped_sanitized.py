"""The C host layer of the products grouped by expert under AddressSanitizer + UndefinedBehaviorSanitizer on the CPU: skl_api_grouped.c with the
sanitizers, everything that would reach the GPU redirected to checking stand-ins (tests/c/host_layer_grouped_check.c). Random orders, products and sums
on host memory, some with allocations refused: what is staged reaches as far as the interface says and no further, every result comes back, nothing
else changes, and no device memory is left."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_host_layer_under_address_and_ub_sanitizers():
    csrc = os.path.join(ROOT, "skl_amd", "csrc")
    built = subprocess.run(["make", "-C", csrc, "../lib/host_layer_grouped_check"], capture_output=True, text=True)
    assert built.returncode == 0, built.stdout[-3000:] + built.stderr[-3000:]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0")
    for args in (["300"], ["300", "0x5EED"]):
        run = subprocess.run([os.path.join(ROOT, "skl_amd", "lib", "host_layer_grouped_check")] + args, capture_output=True, text=True, env=env)
        assert run.returncode == 0, run.stdout[-3000:] + run.stderr[-6000:]
        assert "host layer ok" in run.stdout

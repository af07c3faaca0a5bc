"""What the host layer of the products grouped by expert hands to the kernels where nothing is multiplied (tests/c/host_layer_empty_sums_check.c): no pointer that
the interface leaves open. A kernel that reads through one would fault, so it is looked for on the host."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_a_kernel_finds_no_operand_of_an_empty_sum(tmp_path):
    program = tmp_path / "host_layer_empty_sums_check"
    clang = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "lib", "llvm", "bin", "clang")
    sources = [os.path.join(ROOT, *at) for at in (("skl_amd", "csrc", "skl_api_grouped.c"), ("tests", "c", "host_layer_empty_sums_check.c"))]
    subprocess.run([clang, "-std=c11", "-O1", "-Wall", "-Wextra", "-Werror", *sources, "-o", program], check=True)
    run = subprocess.run([program], capture_output=True, text=True)
    assert run.returncode == 0 and run.stdout == "empty sums ok\n", run.stdout

"""The streaming kernels of the products grouped by expert as they are built, by the rules of test_built_kernels.py: their products are assembly that the compiler does not
look into. Read from the notes and the disassembly of the library's own gfx950 code; no GPU needed."""
import os
import re
import subprocess

import pytest

import test_built_kernels as built
from test_built_kernels import code_objects  # noqa: F401  (a fixture)

GROUPED = re.compile("gemm_grouped_(rows|over)_kernel")
ALL = re.compile("gemm_grouped|gemm_u4|group_rows|group_count")
FEW = re.compile("gemm_grouped_kernel.*ELi2ELi2EE")  # sums with fewer than eight columns, value by value


@pytest.fixture(scope="module")
def kernels(code_objects):  # noqa: F811
    out = {}
    for obj in code_objects:
        text = subprocess.run([os.path.join(built.LLVM, "llvm-objdump"), "-d", "--no-show-raw-insn", obj], check=True, capture_output=True, text=True).stdout
        for part in re.split(r"\n(?=[0-9a-f]{16} <)", text):
            name = re.match(r"[0-9a-f]{16} <([^>]*)>:", part)
            if name and GROUPED.search(name.group(1)):
                out[name.group(1)] = [line.split("//")[0].strip() for line in part.split("\n")[1:] if line.startswith("\t")]
    assert len(out) == 28  # two types: three sizes of tile for two layouts of B; four ways of sums in two sizes
    return out


def test_no_kernel_touches_scratch_memory(code_objects):  # noqa: F811
    seen, bad = 0, []
    for obj in code_objects:
        notes = subprocess.run([os.path.join(built.LLVM, "llvm-readelf"), "--notes", obj], check=True, capture_output=True, text=True).stdout
        for kernel in re.split(r"\n  - \.agpr_count", notes)[1:]:
            value = lambda key: re.search(rf"\.{key}:\s+(\S+)", kernel).group(1)  # noqa: E731
            if ALL.search(value("name")) and not FEW.search(value("name")):
                seen += 1
                if int(value("private_segment_fixed_size")) or int(value("vgpr_spill_count")):
                    bad.append(value("name"))
    assert seen > 60 and not bad, bad


def test_nothing_touches_a_sum_while_its_product_is_under_way(kernels):
    built.test_nothing_touches_a_sum_while_its_product_is_under_way(kernels)


def test_operands_of_a_product_are_written_two_states_ahead(kernels):
    built.test_operands_of_a_product_are_written_two_states_ahead(kernels)


def test_the_loop_is_not_left_with_a_product_under_way(kernels):
    built.test_the_loop_is_not_left_with_a_product_under_way(kernels)


def test_loads_to_lds_are_the_compilers(kernels):
    """It keeps M0 for them, and no assembly here writes it."""
    for name, code in kernels.items():
        loads = [x for x in code if re.match(r"(global_load_lds|buffer_load_\S+ .*\blds\b)", x)]
        assert loads and all(x.startswith("buffer_load") for x in loads), name

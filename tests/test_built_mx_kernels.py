"""The kernels of skl_gemm_mxf4.hip and skl_moe_mxf4.hip whose products are assembly, as they are built: what the compiler does not know of a
product under way, followed along every branch. Read from the disassembly of the library's own gfx950 code; no GPU needed."""
import os
import re
import shutil
import subprocess

import pytest

import skl_amd
from test_built_kernels import LLVM, operands, registers, states

KERNELS = ("gemm_mx_wide_kernel", "moe_in_kernel", "moe_out_kernel")
PASSES = {"16x16x32_bf16": 4, "32x32x64_f8f6f4": 16}  # of four cycles each, of the slowest formats


@pytest.fixture(scope="module")
def objects(tmp_path_factory):
    """(file, its notes) of the code objects that hold these kernels."""
    folder = tmp_path_factory.mktemp("code")
    library = shutil.copy(skl_amd.library_path(), folder / "library.so")
    subprocess.run([os.path.join(LLVM, "llvm-objdump"), "--offloading", library], check=True, cwd=folder, capture_output=True)
    out = []
    for f in sorted(folder.iterdir()):
        if f.name.endswith("gfx950") and f.stat().st_size:
            notes = subprocess.run([os.path.join(LLVM, "llvm-readelf"), "--notes", f], check=True, capture_output=True, text=True).stdout
            if any(name in notes for name in KERNELS):
                out.append((f, notes))
    assert len(out) == 2
    return out


@pytest.fixture(scope="module")
def kernels(objects):
    """Name -> instructions, and for each of them the places that come next."""
    out = {}
    for f, _ in objects:
        text = subprocess.run([os.path.join(LLVM, "llvm-objdump"), "-d", "--no-show-raw-insn", f], check=True, capture_output=True, text=True).stdout
        for part in re.split(r"\n(?=[0-9a-f]{16} <)", text):
            name = re.match(r"[0-9a-f]{16} <([^>]*)>:", part)
            if not name or not any(k in name.group(1) for k in KERNELS):
                continue
            lines = [line.split("//") for line in part.split("\n")[1:] if line.startswith("\t") and "//" in line]
            code = [line[0].strip() for line in lines]
            at = {int(line[1].strip().rstrip(":").split(":")[0], 16): i for i, line in enumerate(lines)}
            places = sorted(at)
            following = []
            for i, instruction in enumerate(code):
                jump = re.match(r"s_(c?branch\w*) (\d+)", instruction)
                nexts = [] if re.match(r"s_(branch|endpgm|setpc)", instruction) else [i + 1]
                if jump:
                    offset = int(jump.group(2))
                    nexts.append(at[places[i] + 4 + 4 * (offset - 65536 if offset >= 32768 else offset)])
                following.append([n for n in nexts if n < len(code)])
            out[name.group(1)] = (code, following)
    assert sum("gemm_mx_wide" in n for n in out) == 2 and sum("moe_" in n for n in out) == 8
    return out


def passes_of(instruction):
    return PASSES[re.match(r"v_mfma_(?:scale_)?f32_(\S+)", instruction).group(1)]


def test_they_touch_no_scratch_memory(objects):
    seen = 0
    for _, notes in objects:
        for kernel in re.split(r"\n  - \.agpr_count", notes)[1:]:
            value = lambda key: re.search(rf"\.{key}:\s+(\S+)", kernel).group(1)
            if any(k in value("name") for k in KERNELS):
                seen += 1
                assert int(value("private_segment_fixed_size")) == 0 and int(value("vgpr_spill_count")) == 0, value("name")
    assert seen == 10


def test_nothing_touches_a_sum_while_its_product_is_under_way(kernels):
    for name, (code, following) in kernels.items():
        for at, instruction in enumerate(code):
            if not instruction.startswith("v_mfma_"):
                continue
            result, latency = registers(operands(instruction)[0]), passes_of(instruction) + 4
            best, todo = {}, [(n, 0) for n in following[at]]
            while todo:
                i, waited = todo.pop()
                if waited >= latency or best.get(i, latency) <= waited:
                    continue
                best[i] = waited
                if not code[i].startswith("v_mfma_"):
                    assert not any(registers(o) & result for o in operands(code[i])), (name, instruction, code[i], waited)
                todo += [(n, waited + states(code[i])) for n in following[i]]


def test_operands_of_a_product_are_written_two_states_ahead(kernels):
    """By vector instructions; what comes from LDS is waited for."""
    for name, (code, following) in kernels.items():
        products = {at: set().union(*(registers(o) for o in operands(x)[1:])) for at, x in enumerate(code) if x.startswith("v_mfma_")}
        assert products
        for at, instruction in enumerate(code):
            if not instruction.startswith("v_") or instruction.startswith(("v_mfma_", "v_cmp", "v_readfirstlane", "v_readlane")):
                continue
            written = registers(operands(instruction)[0]) if operands(instruction) else set()
            todo = [(n, 0) for n in following[at]]
            while todo:
                i, waited = todo.pop()
                if waited >= 2:
                    continue
                assert not (i in products and written & products[i]), (name, instruction, code[i])
                todo += [(n, waited + states(code[i])) for n in following[i]]


def test_every_load_to_lds_has_its_own_m0(kernels):
    for name, (code, _) in kernels.items():
        loads = [at for at, x in enumerate(code) if re.match(r"buffer_load_\S+ .*\blds\b", x)]
        assert loads, name
        for before, at in zip([-1] + loads, loads):
            between = code[before + 1:at]
            assert any(re.match(r"s_\S+ m0,", x) for x in between) and not re.match(r"s_\S+ m0,", between[-1]), (name, code[at - 3:at + 1])

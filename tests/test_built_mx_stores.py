"""Stores of more than two registers in the microscaled 4-bit kernels as they are built: such a store still reads its data two wait states after it is
issued, so no vector instruction may write those registers before. The compiler keeps that distance for its own stores; for those that are assembly it does not
look. Read from the disassembly of the library's own gfx950 code; no GPU needed."""
import os
import re
import shutil
import subprocess

import pytest

import skl_amd
from test_built_kernels import LLVM, operands, registers, states

NAMES = ("gemm_mx_", "moe_", "cvt_to_mx", "cvt_from_mx", "mx_pad")
WIDE_STORE = re.compile(r"(global|flat|buffer)_store_(dwordx[34]|b96|b128)\b")


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """Name -> instructions, and for each of them the places that come next."""
    folder = tmp_path_factory.mktemp("code")
    library = shutil.copy(skl_amd.library_path(), folder / "library.so")
    subprocess.run([os.path.join(LLVM, "llvm-objdump"), "--offloading", library], check=True, cwd=folder, capture_output=True)
    out = {}
    for f in sorted(folder.iterdir()):
        if not f.name.endswith("gfx950") or not f.stat().st_size:
            continue
        notes = subprocess.run([os.path.join(LLVM, "llvm-readelf"), "--notes", f], check=True, capture_output=True, text=True).stdout
        if not any(name in notes for name in NAMES):
            continue
        text = subprocess.run([os.path.join(LLVM, "llvm-objdump"), "-d", "--no-show-raw-insn", f], check=True, capture_output=True, text=True).stdout
        for part in re.split(r"\n(?=[0-9a-f]{16} <)", text):
            name = re.match(r"[0-9a-f]{16} <([^>]*)>:", part)
            if not name or not any(n in name.group(1) for n in NAMES):
                continue
            lines = [line.split("//") for line in part.split("\n")[1:] if line.startswith("\t") and "//" in line]
            code = [line[0].strip() for line in lines]
            places = [int(line[1].strip().split(":")[0], 16) for line in lines]
            at = {place: i for i, place in enumerate(places)}
            following = []
            for i, instruction in enumerate(code):
                jump = re.match(r"s_(c?branch\w*) (\d+)", instruction)
                nexts = [] if re.match(r"s_(branch|endpgm|setpc)", instruction) else [i + 1]
                if jump:
                    offset = int(jump.group(2))
                    nexts.append(at[places[i] + 4 + 4 * (offset - 65536 if offset >= 32768 else offset)])
                following.append([n for n in nexts if n < len(code)])
            out[name.group(1)] = (code, following)
    assert len(out) > 20
    return out


def test_nothing_writes_the_data_of_a_store_on_its_way(kernels):
    seen, past = 0, 0
    for name, (code, following) in kernels.items():
        for at, instruction in enumerate(code):
            if not WIDE_STORE.match(instruction):
                continue
            seen, past = seen + 1, past + instruction.endswith(" nt")
            given = operands(instruction)
            data = registers(given[0] if instruction.startswith("buffer") else given[1])
            assert len(data) >= 3
            todo = [(n, 0) for n in following[at]]
            while todo:
                i, waited = todo.pop()
                if waited >= 2:
                    continue
                vector = code[i].startswith("v_") and not code[i].startswith(("v_cmp", "v_readfirstlane", "v_readlane")) and operands(code[i])
                assert not (vector and registers(operands(code[i])[0]) & data), (name, instruction, code[i], waited)
                todo += [(n, waited + states(code[i])) for n in following[i]]
    assert seen > 50 and past > 10

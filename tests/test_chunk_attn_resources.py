"""What the compiler made of the chunks' attention, from the code built here: no instruction writes a register that a matrix instruction
of the source's own assembly reads as its operand within the next two wait states (the hardware does not wait there by itself, and the compiler
does not look into such assembly), and the registers hold what the loop works on."""

import os
import re
import struct
import subprocess

import pytest

from qwenny_amd.build import LIB
from tests.test_kernel_resources import _kernels

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
needs_build = pytest.mark.skipif(not os.path.exists(LIB), reason="nothing built")


def _code(path, tmp):
    """The gfx950 code objects of the library that name the kernel."""
    with open(path, "rb") as f:
        data = f.read()
    for m in re.finditer(b"__CLANG_OFFLOAD_BUNDLE__", data):
        pos = m.start() + 32
        for _ in range(struct.unpack_from("<Q", data, m.start() + 24)[0]):
            offset, size, n = struct.unpack_from("<QQQ", data, pos)
            elf = data[m.start() + offset:m.start() + offset + size]
            if b"amdgcn" in data[pos + 24:pos + 24 + n] and b"17chunk_attn_kernelI" in elf:
                out = tmp / f"{m.start()}.co"
                out.write_bytes(elf)
                yield str(out)
            pos += 24 + n


def _registers(text):
    return {r for a, b in re.findall(r"\bv\[?(\d+)(?::(\d+))?\]?", text) for r in range(int(a), int(b or a) + 1)}


def _operands(text):
    return re.split(r",(?![^\[]*\])", text)


def too_near(lines):
    """Matrix instructions whose operands were written less than two wait states before, in the order of the listing."""
    found, before = [], []  # (registers written, wait states)
    for line in lines:
        line = line.split("//")[0].strip()
        op, _, rest = line.partition(" ")
        written, states = set(), 1
        if op.startswith("v_mfma"):
            read, passed = set().union(*(_registers(o) for o in _operands(rest)[1:3])), 0
            for regs, n in reversed(before[-2:]):
                if regs & read and passed < 2:
                    found.append(line)
                passed += n
        elif op.startswith("v_") and not op.startswith(("v_cmp", "v_accvgpr_write")):
            written = _registers(_operands(rest)[0])
        elif op == "s_nop":
            states += int(rest, 0)
        before.append((written, states))
    return found


def test_the_search_finds_them():
    mfma = "v_mfma_f32_32x32x16_f16 a[0:15], v[4:7], v[8:11], a[0:15]"
    assert too_near(["v_add_f32_e32 v8, v1, v2", mfma]) and too_near(["v_add_f32_e32 v8, v1, v2", "s_nop 0", mfma])
    assert not too_near(["v_add_f32_e32 v8, v1, v2", "s_nop 1", mfma])
    assert not too_near(["v_add_f32_e32 v8, v1, v2", "s_mov_b32 s0, 0", "s_mov_b32 s0, 0", mfma])
    assert not too_near(["v_add_f32_e32 v12, v1, v2", "v_accvgpr_write_b32 a3, v8", mfma])


@needs_build
@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no disassembler")
def test_operands_are_ready(tmp_path):
    kernels = {}
    for path in _code(LIB, tmp_path):
        listing = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", path], capture_output=True, text=True, check=True).stdout
        for part in re.split(r"\n(?=[0-9a-f]+ <)", listing):
            name = re.match(r"[0-9a-f]+ <(\w+)>:", part)
            if name and "17chunk_attn_kernelI" in name[1]:
                kernels[name[1]] = part.splitlines()[1:]
    assert len(kernels) == 12  # three head sizes, two formats, units of 256 and of 128 rows
    for name, lines in kernels.items():
        assert sum("v_mfma" in line for line in lines) > 20
        assert not too_near(lines), name


@needs_build
@pytest.mark.parametrize("kernel,most", [("chunk_attn_kernel", 64), ("kv_plan_kernel", 0), ("kv_release_kernel", 0), ("kv_fill_kernel", 0),
                                         ("verify_stats_kernel", 0), ("verify_pick_kernel", 0), ("verify_walk_kernel", 0),
                                         ("verify_accept_kernel", 0), ("verify_rest_kernel", 0), ("verify_finish_kernel", 0)])
def test_scratch(kernel, most):
    """None, but for a few numbers of a unit that the widest heads' kernel puts by while its loop runs."""
    found = {n: r for n, r in _kernels(LIB).items() if f"{len(kernel)}{kernel}" in n}
    assert found
    assert max(found.values()) <= most, found

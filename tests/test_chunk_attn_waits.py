"""The waits around the matrix instructions that the chunks' attention writes itself, in the code built here: along every path of the
listing, nothing touches what a product writes before it is through (8 passes and 4 steps), but a product added to it in the same
registers; and nothing that a product starts from was written by a vector instruction less than two steps before. The hardware waits for
neither by itself, and the compiler does not look into such assembly. In the source the first wait has the products' registers as its
operands, so that no reader of them can be moved before it."""

import os
import re
import subprocess

import pytest

from qwenny_amd.build import LIB
from tests.test_chunk_attn_resources import OBJDUMP, _code

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwenny_amd", "csrc", "chunk_attn.hip")
THROUGH, READY = 12, 2  # steps


def _registers(text):
    return {(kind, r) for kind, a, b in re.findall(r"\b([va])\[?(\d+)(?::(\d+))?\]?", text) for r in range(int(a), int(b or a) + 1)}


class Instruction:
    def __init__(self, line):
        text, _, note = line.partition("//")
        self.text = text.strip()
        self.op, _, rest = self.text.partition(" ")
        self.at = int(note.split(":")[0], 16) if note else None
        target = re.search(r"<[^>+]+(?:\+0x([0-9a-f]+))?>", note)
        self.target = int(target[1] or "0", 16) if target and "branch" in self.op else None
        self.product = self.op.startswith("v_mfma")
        operands = re.split(r",(?![^\[]*\])", rest)
        self.parts = [_registers(o) for o in operands]
        self.all = set().union(*self.parts)
        self.written = self.parts[0] if self.op.startswith("v_") and not self.op.startswith("v_cmp") and not self.product else set()
        self.steps = int(rest, 0) + 1 if self.op == "s_nop" else 1


def too_soon(lines):
    """(what wrote, what touches it too soon) of a kernel's listing."""
    code = [Instruction(line) for line in lines if line.strip() and not line.strip().endswith(":")]
    place = {i.at - code[0].at: k for k, i in enumerate(code) if i.at is not None}

    def after(k):
        i = code[k]
        if i.target is not None and i.target in place:
            yield place[i.target]
        if i.op not in ("s_branch", "s_endpgm") and k + 1 < len(code):
            yield k + 1

    found = []
    for k, i in enumerate(code):
        if not i.product and not i.written:
            continue
        most = THROUGH if i.product else READY
        seen, todo = {}, [(n, 0) for n in after(k)]
        while todo:
            n, steps = todo.pop()
            if steps >= most or seen.get(n, most) <= steps:
                continue
            seen[n] = steps
            j = code[n]
            if i.product:
                to = i.parts[0]
                if j.product:  # an addition to the same registers follows without a wait
                    bad = to & (j.parts[1] | j.parts[2]) or any(to & p and to != p for p in (j.parts[0], j.parts[3]))
                else:
                    bad = to & j.all
            else:
                bad = j.product and i.written & (j.parts[1] | j.parts[2] | j.parts[3])
            if bad:
                found.append((i.text, j.text))
            todo += [(m, steps + j.steps) for m in after(n)]
    return found


def _listing(*texts):
    return [f"{t} // {4 * k:012X}: 00000000" for k, t in enumerate(texts)]


FIRST = "v_mfma_f32_32x32x16_f16 v[0:15], v[20:23], v[24:27], 0"
MORE = "v_mfma_f32_32x32x16_f16 v[0:15], v[20:23], v[24:27], v[0:15]"
KEPT = "v_mfma_f32_32x32x16_f16 a[0:15], v[20:23], v[24:27], a[0:15]"
WAIT = ("s_nop 15", "s_nop 3")
READ = "v_fma_f32 v40, v7, v41, v42"


@pytest.mark.parametrize("bad,texts", [
    (0, (FIRST, MORE, *WAIT, READ)), (2, (FIRST, MORE, READ)), (1, (FIRST, "s_nop 10", MORE, READ, *WAIT)),
    (1, (FIRST, "s_nop 9", READ)), (0, (FIRST, "s_nop 11", READ)), (1, (FIRST, "ds_write_b32 v50, v3")),
    (1, (FIRST, "buffer_load_dword v15, v50, s[0:3], 0 offen")), (0, (FIRST, "v_add_f32_e32 v16, v20, v24")),
    (1, (FIRST, "v_mfma_f32_32x32x16_f16 v[100:115], v[12:15], v[24:27], 0")),
    (1, (FIRST, "v_mfma_f32_32x32x16_f16 v[8:23], v[30:33], v[24:27], v[8:23]")),
    (1, (KEPT, "v_accvgpr_read_b32 v3, a9")), (0, (KEPT, *WAIT, "v_accvgpr_read_b32 v3, a9")), (0, (KEPT, "v_add_f32_e32 v9, v9, v9")),
    (1, ("v_accvgpr_write_b32 a3, v60", KEPT)), (0, ("v_accvgpr_write_b32 a3, v60", "s_nop 1", KEPT)),
    (0, ("v_accvgpr_write_b32 a16, v60", KEPT)), (1, ("v_mul_f32_e32 v5, v60, v60", "s_nop 0", MORE)), (1, ("v_mul_f32_e32 v21, v60, v60", KEPT))])
def test_the_search_finds_them(bad, texts):
    assert len(too_soon(_listing(*texts))) == bad, too_soon(_listing(*texts))


def test_the_search_follows_branches():
    """Back over a loop's end, and past what is jumped over."""
    loop = _listing("s_nop 0", READ, *WAIT, FIRST, "s_cbranch_scc1 0")
    loop[-1] += " <kernel+0x4>"
    assert len(too_soon(loop)) == 1
    over = _listing(FIRST, "s_branch 2", *WAIT, READ)
    over[1] += " <kernel+0x10>"
    assert len(too_soon(over)) == 1


def test_waits_hold_the_products_registers():
    """What reads a product's result with the compiler's own instructions does so behind a wait that it depends on."""
    with open(SOURCE) as f:
        text = f.read()
    wait = r'asm volatile\("s_nop 15\\n\\ts_nop 3" : "\+v"\(x\[0\]\)'
    assert re.search(r"products_ready\(f16 \(&x\)\[SETS\]\) \{\s*if constexpr \(SETS == 1\) " + wait + r"\);\s*else " + wait + r', "\+v"\(x\[1\]\)\);', text)
    assert re.search(r"auto first_set = \[&\]\([^)]*\) INLINE \{\s*products_ready\(x\);", text)


@pytest.mark.skipif(not os.path.exists(LIB), reason="nothing built")
@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no disassembler")
def test_nothing_is_touched_too_soon(tmp_path):
    kernels = {}
    for path in _code(LIB, tmp_path):
        listing = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", path], capture_output=True, text=True, check=True).stdout
        for part in re.split(r"\n(?=[0-9a-f]+ <)", listing):
            name = re.match(r"[0-9a-f]+ <(\w+)>:", part)
            if name and "17chunk_attn_kernelI" in name[1]:
                kernels[name[1]] = part.splitlines()[1:]
    assert len(kernels) == 12
    for name, lines in kernels.items():
        found = too_soon(lines)
        assert not found, (name, len(found), found[:3])

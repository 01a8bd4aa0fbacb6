"""The wait states around matrix instructions in the built library. The hardware does not hold a matrix instruction
back for a vector register that a vector instruction has just written, nor another one for a matrix instruction's
result; the compiler spaces out those that it schedules, but does not look into inline assembly. Here every kernel
of the library is walked: along every path
  - two wait states lie between a vector instruction that writes a register and a matrix instruction that reads it;
  - 8 (v_mfma_f32_16x16x32_bf16) or 12 (v_mfma_scale_f32_16x16x128_f8f6f4) lie between a matrix instruction and the
    next other instruction that touches its result.
These are the counts that the compiler keeps for the same instructions by builtins. An instruction is one state,
s_nop n is n + 1."""
import os
import re
import shutil
import struct
import subprocess

import pytest

import gsample

OBJDUMP = shutil.which("llvm-objdump", path="/opt/rocm/llvm/bin")
OPERANDS = 2
RESULT = {"v_mfma_f32_16x16x32_bf16": 8, "v_mfma_scale_f32_16x16x128_f8f6f4": 12}


def registers(operand):
    m = re.match(r"[-|]*([va])(?:(\d+)|\[(\d+):(\d+)\])", operand.strip())
    if not m:
        return set()
    first, last = (m[2], m[2]) if m[2] else (m[3], m[4])
    return {(m[1], i) for i in range(int(first), int(last) + 1)}


class Instruction:
    def __init__(self, name, operands, at, target):
        self.name, self.at, self.target = name, at, target
        self.matrix = name.startswith(("v_mfma", "v_smfma"))
        self.states = int(operands, 0) + 1 if name == "s_nop" else 1
        parts = [registers(p) for p in re.split(r",\s*", operands)]
        vector = name.startswith("v_") and not name.startswith("v_cmp")
        self.written = parts[0] if vector else set()
        if "_swap" in name:
            self.written = parts[0] | parts[1]
        self.read = set().union(*(parts[1:] if self.matrix else parts)) if parts else set()
        self.touched = set().union(*parts)


def kernels(listing):
    """{name: instructions} of a listing."""
    out, here = {}, []
    for line in listing.splitlines():
        m = re.match(r"^[0-9a-f]+ <(.+)>:$", line)
        if m:
            here = out.setdefault(m[1], [])
            continue
        m = re.match(r"^\s+([a-z]\w+)\s*(.*?)\s*// ([0-9A-F]+):", line)
        if m:
            t = re.search(r"<[^>]*\+0x([0-9a-f]+)>\s*$", line)
            here.append(Instruction(m[1], m[2], int(m[3], 16), int(t[1], 16) if t else None))
    return {k: v for k, v in out.items() if v}


def edges(code):
    after = [[] for _ in code]
    place = {i.at - code[0].at: k for k, i in enumerate(code)}
    for k, i in enumerate(code):
        if i.name not in ("s_branch", "s_endpgm", "s_setpc_b64") and k + 1 < len(code):
            after[k].append(k + 1)
        if "branch" in i.name and i.target is not None:
            after[k].append(place[i.target])
    before = [[] for _ in code]
    for k, to in enumerate(after):
        for t in to:
            before[t].append(k)
    return before, after


def too_near(code, start, steps, need, wrong):
    """Whether an instruction that `wrong` names comes before `need` wait states have passed."""
    todo, seen = [(k, 0) for k in steps[start]], set()
    while todo:
        k, passed = todo.pop()
        if wrong(code[k]):
            return True
        passed += code[k].states
        if passed < need and (k, passed) not in seen:
            seen.add((k, passed))
            todo += [(n, passed) for n in steps[k]]
    return False


def faults(code):
    before, after = edges(code)
    for k, i in enumerate(code):
        if not i.matrix:
            continue
        if too_near(code, k, before, OPERANDS, lambda o: not o.matrix and o.written & i.read):
            yield f"{i.at:x}: {i.name} reads what was just written"
        need = RESULT.get(i.name, 0)
        if need and too_near(code, k, after, need, lambda o: not o.matrix and o.touched & i.written):
            yield f"{i.at:x}: the result of {i.name} is touched too soon"


def code_objects(library):
    """The gfx950 code objects in a library built by hipcc."""
    with open(library, "rb") as f:
        data = f.read()
    at = data.find(b"__CLANG_OFFLOAD_BUNDLE__")
    while at >= 0:
        (count,) = struct.unpack_from("<Q", data, at + 24)
        entry = at + 32
        for _ in range(count):
            offset, size, length = struct.unpack_from("<QQQ", data, entry)
            if b"gfx950" in data[entry + 24:entry + 24 + length]:
                yield data[at + offset:at + offset + size]
            entry += 24 + length
        at = data.find(b"__CLANG_OFFLOAD_BUNDLE__", at + 24)


LISTING = """
0000000000000100 <k>:
\tv_lshlrev_b32_e32 v9, v1, v9                               // 000000000100: 00000000
{between}
\tv_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[10:13], v[20:27], a[0:3], v9, v8 op_sel_hi:[0,0,0] cbsz:4// 000000000120: 0
\ts_nop {nop}                                                // 000000000130: 00000000
\tv_accvgpr_read_b32 v1, a2                                  // 000000000134: 00000000
\ts_endpgm                                                   // 000000000138: 00000000
"""


@pytest.mark.parametrize("between,nop,want", [
    ("\ts_nop 1 // 000000000104: 0", 11, 0),
    ("\ts_nop 0 // 000000000104: 0", 11, 1),
    ("\tv_mov_b32_e32 v30, v9 // 000000000104: 0", 15, 1),
    ("\tv_mov_b32_e32 v30, v9 // 000000000104: 0\n\ts_nop 0 // 000000000108: 0", 10, 1),
    ("\ts_nop 0 // 000000000104: 0", 3, 2),
])
def test_the_walk_sees_short_waits(between, nop, want):
    code = kernels(LISTING.format(between=between, nop=nop))["k"]
    assert len(list(faults(code))) == want


@pytest.mark.skipif(OBJDUMP is None, reason="llvm-objdump is not installed")
def test_every_matrix_instruction_of_the_library_has_its_waits(tmp_path):
    gsample.library()
    found, matrix = [], 0
    for n, data in enumerate(code_objects(gsample.runtime.LIB_PATH)):
        path = os.path.join(tmp_path, f"{n}.o")
        with open(path, "wb") as f:
            f.write(data)
        text = subprocess.run([OBJDUMP, "-d", "--mcpu=gfx950", path], check=True, capture_output=True, text=True).stdout
        for name, code in kernels(text).items():
            matrix += sum(i.matrix for i in code)
            found += [f"{name} {f}" for f in faults(code)]
    assert matrix > 1000  # (the library's products were seen)
    assert not found, (len(found), found[:5])

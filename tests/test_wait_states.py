"""The wait states that gfx950 leaves to the software, in the code that was built.

The hardware does not hold back an instruction for some of the results that it
reads.  The compiler puts s_nop between its own instructions, but sees neither
into nor across inline assembly, which the loads into LDS and some matrix
products of this library are.  Checked here over every path of every kernel in
the built library's disassembly:

* M0 written by a scalar instruction -> a load into LDS, which takes its LDS
  address from it: 1 wait state.
* A scalar register written by a vector instruction (v_readfirstlane) -> a memory
  instruction that takes its address from it: 5.
* A register written by a vector instruction -> a matrix instruction that reads
  it, as operand, scale or accumulator: 2.
* A matrix instruction's result -> anything but a matrix instruction: 5 for the
  shortest of them, 3 more for one of 16 x 16 x 128 or 32 x 32.

Every instruction is one wait state, s_nop n is n + 1; what an instruction waits
for by itself (memory, LDS) is not counted on.
"""
import re
import struct
import subprocess
from pathlib import Path

import pytest

from conftest import LIB_PATH

OBJDUMP = Path("/opt/rocm/llvm/bin/llvm-objdump")
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def code_objects(path):
    """The gfx950 code objects in a host library."""
    data = path.read_bytes()
    at = data.find(MAGIC)
    while at >= 0:
        count, = struct.unpack_from("<Q", data, at + len(MAGIC))
        p = at + len(MAGIC) + 8
        for _ in range(count):
            offset, size, name = struct.unpack_from("<QQQ", data, p)
            if size and b"gfx950" in data[p + 24:p + 24 + name]:
                yield data[at + offset:at + offset + size]
            p += 24 + name
        at = data.find(MAGIC, at + 1)


REG = re.compile(r"\b([av])(?:(\d+)\b|\[(\d+):(\d+)\])")
SCALAR = re.compile(r"\bs(?:(\d+)\b|\[(\d+):(\d+)\])")
LINE = re.compile(r"^\t(\S+)\s*(.*?)\s*// ([0-9A-F]{12}):")
TARGET = re.compile(r"<[^<>]*?(?:\+0x([0-9a-f]+))?>\s*$")


def registers(text):
    """The vector and accumulation registers that `text` names, as (kind, number)."""
    out = set()
    for kind, one, lo, hi in REG.findall(text):
        out.update((kind, n) for n in (range(int(one), int(one) + 1) if one else range(int(lo), int(hi) + 1)))
    return out


def scalars(text):
    """The scalar registers that `text` names."""
    out = set()
    for one, lo, hi in SCALAR.findall(text):
        out.update(range(int(one), int(one) + 1) if one else range(int(lo), int(hi) + 1))
    return out


class Instruction:
    __slots__ = ("name", "text", "states", "before", "after")

    def __init__(self, name, text):
        self.name, self.text = name, text
        self.states = int(text, 0) + 1 if name == "s_nop" else 1
        self.before, self.after = [], []

    @property
    def args(self):
        return [a.strip() for a in re.split(r",(?![^\[]*\])", self.text)]

    @property
    def matrix(self):
        return self.name.startswith(("v_mfma", "v_smfma"))

    @property
    def into_lds(self):
        return "load_lds" in self.name or (self.name.startswith("buffer_load") and " lds" in self.text)

    @property
    def memory(self):
        return self.name.startswith(("global_", "buffer_", "flat_", "scratch_"))

    @property
    def writes(self):
        """Registers that a vector instruction writes."""
        if "swap" in self.name:
            return registers(self.text)
        return registers(self.args[0])

    @property
    def reads(self):
        return registers(",".join(self.args[1:]))


def kernels(disassembly):
    """(name, instructions) of each function, linked along its paths."""
    name, code, at, start = None, [], {}, 0

    def linked():
        for i, ins in enumerate(code):
            ends = ins.name in ("s_endpgm", "s_branch", "s_setpc_b64")
            nexts = [] if ends or i + 1 == len(code) else [i + 1]
            if ins.name.startswith(("s_branch", "s_cbranch")):
                m = TARGET.search(ins.text)
                assert m, ins.text
                nexts.append(at[start + int(m.group(1) or "0", 16)])
            for n in nexts:
                ins.after.append(code[n])
                code[n].before.append(ins)
        return name, code

    for line in disassembly.splitlines():
        if line.endswith(">:"):
            if code:
                yield linked()
            name, code, at, start = line[1:-2], [], {}, None
            continue
        m = LINE.match(line)
        if m:
            where = int(m.group(3), 16)
            start = where if start is None else start
            at[where] = len(code)
            text = m.group(2)
            if m.group(1).startswith(("s_branch", "s_cbranch")):
                text = line[line.index("//"):].rstrip()
            code.append(Instruction(m.group(1), text))
    if code:
        yield linked()


def near(ins, side, states):
    """Instructions with fewer than `states` wait states between them and `ins`,
    on any path before or after it."""
    todo, seen = [(n, states) for n in getattr(ins, side)], {}
    while todo:
        n, left = todo.pop()
        if seen.get(id(n), 0) >= left:
            continue
        if id(n) not in seen:
            yield n, states - left
        seen[id(n)] = left
        if left > n.states:
            todo += [(m, left - n.states) for m in getattr(n, side)]


def missing_waits(code):
    found = []
    for ins in code:
        if ins.into_lds:
            found += [("M0 -> load into LDS", n, ins, gap) for n, gap in near(ins, "before", 1)
                      if n.name.startswith("s_") and n.args[0] == "m0"]
        if ins.memory and (address := scalars(ins.text)):
            found += [("vector -> address", n, ins, gap) for n, gap in near(ins, "before", 5)
                      if n.name.startswith("v_") and not n.matrix and scalars(n.args[0]) & address]
        if ins.matrix:
            reads, result = ins.reads, registers(ins.args[0])
            found += [("vector -> matrix", n, ins, gap) for n, gap in near(ins, "before", 2)
                      if n.name.startswith("v_") and not n.matrix and n.writes & reads]
            wide = "16x16x128" in ins.name or "32x32" in ins.name
            found += [("matrix -> other", ins, n, gap) for n, gap in near(ins, "after", 8 if wide else 5)
                      if not n.matrix and registers(n.text) & result]
    return found


def test_the_check_sees_missing_waits():
    """The check itself, on code that lacks a wait: next to each other, behind a
    branch, around a loop; and on the same code with the wait."""
    def listing(*body):
        out, pc = ["0 <k>:"], 0
        for text in body:
            ins, _, to = text.partition(" @")
            out.append(f"\t{ins} // {pc:012X}: 00000000" + (f" <k+0x{4 * int(to):x}>" if to else ""))
            pc += 4
        (_, code), = kernels("\n".join(out).replace("0 <k>:", "<k>:"))
        return [kind for kind, *_ in missing_waits(code)]

    load, m0 = "global_load_lds_dwordx4 v0, s[2:3]", "s_mov_b32 m0, s4"
    assert listing(m0, load, "s_endpgm") == ["M0 -> load into LDS"]
    assert listing(m0, "s_nop 0", load, "s_endpgm") == []
    assert listing("v_readfirstlane_b32 s3, v1", "s_nop 3", load, "s_endpgm") == ["vector -> address"]
    assert listing("v_readfirstlane_b32 s3, v1", "s_nop 4", load, "s_endpgm") == []
    mfma = "v_mfma_scale_f32_16x16x128_f8f6f4 a[4:7], v[8:11], v[12:15], a[4:7], v1, v2 op_sel_hi:[0,0,0] cbsz:4 blgp:4"
    for write in ("v_accvgpr_write_b32 a5, 0", "v_mov_b32_e32 v15, v3", "v_mov_b32_e32 v2, 0",
                  "v_permlane32_swap_b32_e32 v90, v8"):
        assert listing(write, mfma, "s_endpgm") == ["vector -> matrix"]
        assert listing(write, "s_waitcnt lgkmcnt(0)", mfma, "s_endpgm") == ["vector -> matrix"]
        assert listing(write, "s_nop 1", mfma, "s_endpgm") == []
    assert listing("s_nop 0", mfma, "v_mov_b32_e32 v1, 0", "s_cbranch_scc1 1 @1", "s_endpgm") == ["vector -> matrix"]
    assert listing("v_mov_b32_e32 v7, 0", mfma, "s_endpgm") == []
    read = "v_accvgpr_read_b32 v0, a7"
    assert listing(mfma, "s_nop 6", read, "s_endpgm") == ["matrix -> other"]
    assert listing(mfma, "s_nop 7", read, "s_endpgm") == []
    assert listing(mfma, mfma, "s_nop 7", read, "s_endpgm") == []


@pytest.mark.skipif(not OBJDUMP.exists(), reason="no llvm-objdump")
def test_no_wait_state_is_missing_in_the_built_kernels(tmp_path):
    if not LIB_PATH.exists():
        pytest.fail(f"{LIB_PATH} missing: run __graft_entry__.build() first")
    found, loads, matrix = [], 0, 0
    for i, obj in enumerate(code_objects(LIB_PATH)):
        path = tmp_path / f"{i}.co"
        path.write_bytes(obj)
        text = subprocess.run([OBJDUMP, "-d", "--no-leading-addr", path], check=True, capture_output=True, text=True).stdout
        for name, code in kernels(text):
            loads += sum(ins.into_lds for ins in code)
            matrix += sum(ins.matrix for ins in code)
            found += [f"{name}: {kind}, {gap} wait states: {a.name} {a.text} ... {b.name} {b.text}"
                      for kind, a, b, gap in missing_waits(code)]
    assert loads > 1000 and matrix > 1000  # the library was really taken apart
    assert not found, f"{len(found)} missing waits, first: " + "\n".join(found[:5])

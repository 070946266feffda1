"""The built library's code: no instruction touches a matrix instruction's result before it is there, and no load to
LDS reads m0 before it is written.

The processor does not wait by itself between a matrix instruction and a vector, memory or LDS instruction that
touches the registers it writes; the compiler leaves room for it.  This walks every path behind every matrix
instruction of the built kernels, over branches too, and counts the instructions until its result is touched.  A
place that is too near reads what was in the registers before, now and then.

Wait states after an instruction of n passes (gfx950): n + 4 until its result may be read or written, n + 2 for
those that multiply fp32, n - 1 until registers that it only adds from may be overwritten.  (In the code between two
branches the compiler keeps to these numbers everywhere.)

A load from memory to LDS takes its place there from m0, one state after a scalar instruction wrote it at the
earliest; and its address from scalar registers, five states after a vector instruction wrote them.  In assembly
written by hand the compiler sees to neither.
"""
import re
import shutil
import struct
import subprocess

import pytest

from llmcompressor_amd import _lib

PASSES = {"16x16x32_bf16": 4, "16x16x32_f16": 4, "32x32x16_bf16": 8, "32x32x16_f16": 8, "16x16x4_f32": 8, "32x32x2_f32": 16}
BUNDLE = b"__CLANG_OFFLOAD_BUNDLE__"
REGISTERS = re.compile(r"\b([va])(?:(\d+)\b|\[(\d+):(\d+)\])")
OBJDUMP = shutil.which("llvm-objdump", path="/opt/rocm/llvm/bin") or shutil.which("llvm-objdump")


def code_objects(data: bytes):
    """The gfx950 code objects bundled in a library."""
    at = data.find(BUNDLE)
    while at >= 0:
        (count,), p = struct.unpack_from("<Q", data, at + 24), at + 32
        for _ in range(count):
            offset, size, n = struct.unpack_from("<3Q", data, p)
            if b"gfx950" in data[p + 24:p + 24 + n] and size:
                yield data[at + offset:at + offset + size]
            p += 24 + n
        at = data.find(BUNDLE, at + 24)


def registers(text: str) -> frozenset:
    out = set()
    for kind, one, first, last in REGISTERS.findall(text):
        out.update((kind, i) for i in (range(int(one), int(one) + 1) if one else range(int(first), int(last) + 1)))
    return frozenset(out)


class Instruction:
    def __init__(self, op: str, operands: str, target: int | None):
        self.op, self.target = op, target
        self.states = int(operands, 0) + 1 if op == "s_nop" else 1
        parts = re.split(r",\s*(?![^\[]*\])", operands)
        self.all, self.first = registers(operands), registers(parts[0])
        self.matrix = PASSES.get(op.partition("mfma_f32_")[2].removesuffix("_e64")) if "mfma" in op else None
        if "mfma" in op:
            assert self.matrix, f"{op}: how many passes does it take?"
            self.read, self.added = registers(",".join(parts[1:3])), registers(parts[3].split()[0])
        self.ends = op in ("s_endpgm", "s_branch") or op.startswith("s_setpc")


def parse(lines):
    """(instructions, index of each address) of a function's listing."""
    code, at = [], {}
    for line in lines:
        text, _, comment = line.partition("//")
        text = text.strip()
        address = re.match(r"\s*([0-9A-Fa-f]+):", comment)
        if not text or not address:
            continue
        op, _, operands = text.partition(" ")
        target = None
        if op.startswith("s_cbranch") or op == "s_branch":
            # in words of four bytes from the next instruction on
            jump = int(operands.split()[0], 0)
            target = int(address[1], 16) + 4 + 4 * (jump - 65536 if jump > 32767 else jump)
        at[int(address[1], 16)] = len(code)
        code.append(Instruction(op, operands, target))
    return code, at


def functions(listing):
    """(name, instructions, index of each address) of every function that has matrix instructions."""
    name, lines = None, []
    for line in listing:
        head = re.match(r"^[0-9a-f]+ <(.*)>:", line)
        if head:
            if any("mfma" in s for s in lines):
                yield name, *parse(lines)
            name, lines = head[1], []
        else:
            lines.append(line)
    if any("mfma" in s for s in lines):
        yield name, *parse(lines)


def too_near(code, at):
    """(matrix instruction, what comes too near behind it, wait states, those needed), by index."""
    found = []
    for m, first in enumerate(code):
        if first.matrix is None:
            continue
        fp32 = first.op.removesuffix("_e64").endswith("x2_f32") or first.op.removesuffix("_e64").endswith("x4_f32")
        for result, need, live in ((True, first.matrix + (2 if fp32 else 4), first.first),
                                   (False, first.matrix - 1, first.added - first.first)):
            paths, seen = [(m + 1, 0, live)], {}
            while paths:
                i, states, live = paths.pop()
                while live and states < need and i < len(code):
                    c = code[i]
                    if c.matrix is not None:
                        if result and c.read & live:
                            found.append((m, i, states, need))
                        live = live - c.first
                    else:
                        hit = (c.all if result else c.first) & live
                        if hit:
                            found.append((m, i, states, need))
                            live = live - hit
                    states += c.states
                    if c.target is not None and states < seen.get((c.target, live), need):
                        seen[c.target, live] = states
                        paths.append((at[c.target], states, live))
                    if c.ends:
                        break
                    i += 1
    return found


SCALARS = re.compile(r"\bs(?:(\d+)\b|\[(\d+):(\d+)\])")


def scalars(text: str) -> set:
    return {i for one, first, last in SCALARS.findall(text)
            for i in (range(int(one), int(one) + 1) if one else range(int(first), int(last) + 1))}


def early_loads(listing):
    """(function, what wrote m0 or a scalar of the address too near before, the load to LDS)"""
    name, before = None, []
    for line in listing:
        head = re.match(r"^[0-9a-f]+ <(.*)>:", line)
        if head:
            name, before = head[1], []
            continue
        op, _, operands = line.partition("//")[0].strip().partition(" ")
        if not op:
            continue
        if "load_lds" in op:
            states, address = 0, scalars(operands)
            for last, written, took in reversed(before):
                if states < 1 and last.startswith("s_") and written.strip() == "m0":
                    yield name, f"{last} {written}", op
                if states < 5 and last.startswith("v_") and scalars(written) & address:
                    yield name, f"{last} {written}", op
                states += took
        before = [*before[-5:], (op, operands.split(",")[0], int(operands, 0) + 1 if op == "s_nop" else 1)]


def test_early_loads_are_found():
    wait = "\ts_nop 0  // 1: 0"
    load = "\tglobal_load_lds_dwordx4 v1, s[4:5]  // 1: 0"
    head = "0000000000001000 <kernel>:"
    m0, base = "\ts_mov_b32 m0, s7  // 1: 0", "\tv_readfirstlane_b32 s5, v3  // 1: 0"
    assert [f[1] for f in early_loads([head, m0, load])] == ["s_mov_b32 m0"]
    assert not list(early_loads([head, m0, wait, load]))
    assert [f[1] for f in early_loads([head, base, m0, wait, wait, wait, load])] == ["v_readfirstlane_b32 s5"]
    assert not list(early_loads([head, base, m0, *[wait] * 4, load]))


def test_walk_finds_what_a_branch_hides():
    """Results read three states behind their instruction on one of two paths, eight on the other."""
    def listing(pad):
        lines = ["0000000000001000 <kernel>:"]
        ops = ["v_mfma_f32_16x16x32_bf16 a[4:7], v[0:3], v[4:7], a[0:3]", "s_cbranch_vccnz 6",
               *["v_mov_b32_e32 v9, v10"] * 5, "s_branch 1", f"s_nop {pad}", "v_accvgpr_read_b32 v12, a3",
               "v_accvgpr_read_b32 v12, a7", "s_endpgm"]
        sizes = [8, *[4] * 10, 4]
        address = 0x1000
        for op, size in zip(ops, sizes):
            lines.append(f"\t{op}  // {address:012X}: 00000000")
            address += size
        return lines

    # a branch, s_nop 0 and the read of a3: 3 states
    (_, code, at), = functions(listing(0))
    assert [(code[i].op, s, n) for _, i, s, n in too_near(code, at)] == [("v_accvgpr_read_b32", 3, 8)]
    (_, code, at), = functions(listing(5))
    assert not too_near(code, at)


@pytest.mark.skipif(OBJDUMP is None or not _lib.LIB_PATH.exists(), reason="needs llvm-objdump and the built library")
def test_built_code_waits(tmp_path):
    objects = list(code_objects(_lib.LIB_PATH.read_bytes()))
    assert objects
    seen, near, early = 0, [], []
    for n, o in enumerate(objects):
        path = tmp_path / f"{n}.co"
        path.write_bytes(o)
        listing = subprocess.run([OBJDUMP, "-d", "--mcpu=gfx950", str(path)], stdout=subprocess.PIPE, text=True,
                                 check=True).stdout.splitlines()
        early += early_loads(listing)
        for name, code, at in functions(listing):
            seen += 1
            found = too_near(code, at)
            if found:
                near.append((name, len(found), [(code[m].op, code[i].op, s, need) for m, i, s, need in found[:3]]))
    assert seen > 100
    assert not near, f"{len(near)} kernels touch results too early: {near[:5]}"
    assert not early, f"{len(early)} loads to LDS come too early: {early[:5]}"

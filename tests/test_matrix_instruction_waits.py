"""The wait states around the matrix instructions and loads that the kernels write out.

The products write their matrix instructions out (the compiler would move the accumulators
about) and their loads into LDS, so the compiler does not see them and puts no waits between
them and its own instructions: that none are missing depends on the registers it chose.  Here
the library's code is disassembled and every path through each kernel followed:

* a vector register written by a vector instruction is read by a matrix instruction (as an
  operand, an accumulator or a scale) two wait states later at the earliest;
* a matrix instruction's results are touched by anything but a matrix instruction that
  adds to just those 12 wait states later at the earliest, what the longest of
  those used here (e4m3: 32 cycles, 8 passes) asks for; some of them, or as an operand, not
  before that either;
* a scalar register written by a vector instruction (readfirstlane, a comparison) is read by
  a memory instruction five wait states later at the earliest;
* m0 is written by the written-out loads only: they do not tell the compiler, for which it is
  a reserved register, and which has no use of its own for it in these kernels.

An instruction is one wait state, ``s_nop n`` is n + 1.
"""

import re
import struct
import subprocess
from pathlib import Path

import pytest

from offload_adam_amd import _build

OBJDUMP = Path("/opt/rocm/llvm/bin/llvm-objdump")
AFTER_VECTOR, AFTER_MATRIX, AFTER_SCALAR = 2, 12, 5
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def code_objects(library):
    """The gfx950 code objects that a host library carries."""
    data = library.read_bytes()
    at = data.find(MAGIC)
    while at >= 0:
        count, = struct.unpack_from("<Q", data, at + len(MAGIC))
        entry = at + len(MAGIC) + 8
        for _ in range(count):
            offset, size, name = struct.unpack_from("<QQQ", data, entry)
            if _build.OFFLOAD_ARCH.encode() in data[entry + 24:entry + 24 + name] and size:
                yield data[at + offset:at + offset + size]
            entry += 24 + name
        at = data.find(MAGIC, at + 1)


def kernels(text):
    """Name and instructions (address, mnemonic, operands, branch target) of each function."""
    name, code = None, []
    for line in text.splitlines():
        head = re.match(r"^[0-9a-f]+ <(.+)>:$", line)
        if head:
            if name:
                yield name, code
            name, code = head[1], []
            continue
        m = re.match(r"^\s+(\S+)(?:\s+(.*?))?\s*// ([0-9A-F]+):.*?(?:<.*\+0x([0-9a-f]+)>)?\s*$", line)
        if m and name:
            code.append((int(m[3], 16), m[1], m[2] or "", m[4]))
    if name:
        yield name, code


def registers(token):
    token = token.strip().lstrip("-|").rstrip("|")
    m = re.match(r"^([vas])\[(\d+):(\d+)\]", token)
    if m:
        return frozenset((m[1], i) for i in range(int(m[2]), int(m[3]) + 1))
    m = re.match(r"^([vas])(\d+)\b", token)
    return frozenset([(m[1], int(m[2]))]) if m else frozenset()


def scalar(r):
    return r[0] == "s"


def parsed(op, operands):
    """(kind, registers read, registers written, accumulator)"""
    args = [registers(a) for a in re.split(r",\s*(?![^\[]*\])", operands)] if operands else []
    none = frozenset()
    if op.startswith("v_mfma"):
        return "matrix", none.union(*args[1:]), args[0], args[3]
    read = none.union(*args) if args else none  # a written register counts as touched
    if op.startswith("v_"):
        # comparisons of the long form write scalar registers, additions with carry both
        written = args[0] | frozenset(r for r in (args[1] if len(args) > 1 and "_co_" in op else ())
                                      if scalar(r)) if args else none
        return "vector", read, written, none
    memory = op.startswith(("buffer_", "global_", "flat_", "scratch_"))
    return "memory" if memory else "other", read, none, none


def missing_waits(code):
    """Instructions that come too early, with what they are too early for."""
    if not any(op.startswith("v_mfma") for _, op, _, _ in code):
        return []
    base = code[0][0]
    index = {a: i for i, (a, _, _, _) in enumerate(code)}
    info = [parsed(op, args) for _, op, args, _ in code]
    length = [int(args, 0) + 1 if op == "s_nop" else 1 for _, op, args, _ in code]
    found, seen, todo = {}, {}, [(0, {}, {})]
    starts = {0} | {index[base + int(t, 16)] for _, _, _, t in code if t}
    starts |= {i + 1 for i, (_, op, _, _) in enumerate(code) if "branch" in op}

    def merge(i, vector, matrix):
        old = seen.get(i)
        if old is None:
            seen[i] = (dict(vector), dict(matrix))
            return True
        grew = False
        for have, new in zip(old, (vector, matrix)):
            for r, age in new.items():
                if age < have.get(r, (99,)):
                    have[r] = age
                    grew = True
        return grew

    while todo:
        i, vector, matrix = todo.pop()
        first = True
        while i < len(code):
            if (i in starts or first) and not merge(i, vector, matrix):
                break
            if i in starts or first:
                vector, matrix = dict(seen[i][0]), dict(seen[i][1])
            first = False
            _, op, args, target = code[i]
            kind, read, written, acc = info[i]
            if kind == "matrix":
                for r in read:
                    if vector.get(r, (99,))[0] < AFTER_VECTOR:
                        found.setdefault(i, vector[r][1])
                    if r in matrix and matrix[r][0] < AFTER_MATRIX and not (
                            r in acc and matrix[r][2] == acc):
                        found.setdefault(i, matrix[r][1])
                for r in written:
                    if r in matrix and matrix[r][0] < AFTER_MATRIX and matrix[r][2] != written:
                        found.setdefault(i, matrix[r][1])
            else:
                for r in read | written:
                    if r in matrix and matrix[r][0] < AFTER_MATRIX:
                        found.setdefault(i, matrix[r][1])
                    if kind == "memory" and scalar(r) and r in vector:
                        found.setdefault(i, vector[r][1])
            step = length[i]
            vector = {r: (a + step, j) for r, (a, j) in vector.items()
                      if a + step < (AFTER_SCALAR if scalar(r) else AFTER_VECTOR)}
            matrix = {r: (a + step, j, w) for r, (a, j, w) in matrix.items()
                      if a + step < AFTER_MATRIX}
            for r in written:
                if kind == "matrix":
                    matrix[r] = (0, i, written)
                elif kind == "vector":
                    vector[r] = (0, i)
            if op == "s_endpgm":
                break
            if target is not None and "branch" in op:
                todo.append((index[base + int(target, 16)], dict(vector), dict(matrix)))
                if op == "s_branch":
                    break
            i += 1
    return [(f"{code[i][1]} {code[i][2]}", f"{code[j][1]} {code[j][2]}") for i, j in sorted(found.items())]


def listing(*lines):
    """A kernel of these lines, as the disassembler prints it; `@n` is line n."""
    out = ["0000000000001000 <k>:"]
    for i, line in enumerate(lines):
        to = re.search(r"@(\d+)", line)
        end = f" <k+0x{int(to[1]) * 4:x}>" if to else ""
        out.append(f"\t{line.replace('@', '')}  // {0x1000 + 4 * i:012X}: 00000000{end}")
    (_, code), = kernels("\n".join(out))
    return code


MFMA = "v_mfma_f32_16x16x32_bf16 a[0:3], v[4:7], v[8:11], a[0:3]"


@pytest.mark.parametrize("lines, expected", [
    ((MFMA, MFMA, "s_endpgm"), 0),
    (("v_mov_b32_e32 v4, v20", MFMA, "s_endpgm"), 1),
    (("v_mov_b32_e32 v4, v20", "s_nop 0", MFMA, "s_endpgm"), 1),
    (("v_mov_b32_e32 v4, v20", "s_nop 1", MFMA, "s_endpgm"), 0),
    (("v_accvgpr_write_b32 a3, v20", "s_mov_b32 s1, 0", MFMA, "s_endpgm"), 1),
    (("v_mov_b32_e32 v20, v4", MFMA, "s_endpgm"), 0),
    ((MFMA, "s_nop 10", "v_accvgpr_read_b32 v1, a0", "s_endpgm"), 1),
    ((MFMA, "s_nop 10", "s_nop 0", "v_accvgpr_read_b32 v1, a0", "s_endpgm"), 0),
    ((MFMA, "s_nop 3", "scratch_store_dwordx4 off, a[0:3], s32 offset:16", "s_endpgm"), 1),
    ((MFMA, "s_nop 3", "v_accvgpr_write_b32 a2, v1", "s_endpgm"), 1),
    ((MFMA, "s_nop 3", "v_mfma_f32_16x16x32_bf16 a[2:5], v[4:7], v[8:11], a[2:5]", "s_endpgm"), 1),
    (("v_readfirstlane_b32 s8, v1", "s_nop 3", "buffer_load_dword v2, s[8:11], 0 offen lds"), 1),
    (("v_readfirstlane_b32 s8, v1", "s_nop 4", "buffer_load_dword v2, s[8:11], 0 offen lds"), 0),
    (("s_mov_b32 s8, s1", "buffer_load_dword v2, s[8:11], 0 offen lds"), 0),
    (("v_cmp_gt_i32_e64 s[10:11], s2, v1", "buffer_load_dword v2, s[8:11], 0 offen lds"), 1),
    (("v_add_co_u32_e64 v1, s[8:9], v2, v3", "buffer_load_dword v2, s[8:11], 0 offen lds"), 1),
    # round a loop, and past a branch
    ((MFMA, "v_mov_b32_e32 v8, v1", "s_cbranch_scc1 @0", "s_endpgm"), 1),
    ((MFMA, "v_mov_b32_e32 v8, v1", "s_nop 1", "s_cbranch_scc1 @0", "s_endpgm"), 0),
    (("v_mov_b32_e32 v8, v1", "s_cbranch_scc1 @4", "s_nop 1", "s_nop 1", MFMA, "s_endpgm"), 1),
    (("v_mov_b32_e32 v8, v1", "s_branch @4", "s_nop 1", "s_nop 1", MFMA, "s_endpgm"), 1),
    (("s_branch @3", "v_mov_b32_e32 v8, v1", "s_branch @5", MFMA, "s_endpgm", MFMA, "s_endpgm"), 0),
    (("v_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[4:11], v[12:19], a[0:3], v20, v21 "
      "op_sel_hi:[0,0,0]", "s_endpgm"), 0),
    (("v_mov_b32_e32 v21, v1", "v_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[4:11], v[12:19], "
      "a[0:3], v20, v21 op_sel_hi:[0,0,0]", "s_endpgm"), 1),
])
def test_the_check_itself(lines, expected):
    assert len(missing_waits(listing(*lines, MFMA, "s_endpgm"))) == expected


@pytest.fixture(scope="module")
def library(tmp_path_factory):
    """Name and code of every kernel with matrix instructions."""
    assert _build.LIB_PATH.exists(), "build the library first"
    out = []
    for i, blob in enumerate(code_objects(_build.LIB_PATH)):
        file = tmp_path_factory.mktemp("code") / f"{i}.co"
        file.write_bytes(blob)
        text = subprocess.run([OBJDUMP, "-d", str(file)], capture_output=True, text=True,
                              check=True).stdout
        out += [(name, code) for name, code in kernels(text)
                if any(op.startswith("v_mfma") for _, op, _, _ in code)]
    assert len(out) > 50
    return out


def test_no_wait_is_missing(library):
    for name, code in library:
        early = missing_waits(code)
        assert not early, f"{name}: {len(early)}, first {early[0]}"


def test_m0_is_the_loads_own(library):
    written = 0
    for name, code in library:
        for i, (_, op, args, _) in enumerate(code):
            if re.search(r"\bm0\b", args):
                assert op == "s_mov_b32" and args.startswith("m0, s"), f"{name}: {op} {args}"
                # a wait state, or the matrix instruction that the load goes with
                assert code[i + 1][1].startswith(("s_nop", "v_mfma")), name
                assert code[i + 2][1].startswith("buffer_load") and "lds" in code[i + 2][2], name
                written += 1
    assert written > 500

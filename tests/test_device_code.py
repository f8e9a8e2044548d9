"""What the compiler cannot check in the kernels' own assembly statements, read off the sources and off the device code that
was built from them."""
import re
import shutil
import struct
import subprocess
from pathlib import Path

import pytest

from int4linear_amd import build

OBJDUMP = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def code_objects(library: bytes):
    """The gfx950 code objects in a library: (offset, size, name) entries behind the magic of every bundle."""
    at = library.find(MAGIC)
    while at >= 0:
        pos = at + len(MAGIC)
        (count,) = struct.unpack_from("<Q", library, pos)
        pos += 8
        for _ in range(count if count < 16 else 0):
            offset, size, length = struct.unpack_from("<QQQ", library, pos)
            name = library[pos + 24 : pos + 24 + length]
            pos += 24 + length
            if name.endswith(b"gfx950") and size:
                yield library[at + offset : at + offset + size]
        at = library.find(MAGIC, at + 1)


def scalar_registers(operands: str):
    out = {"vcc"} if "vcc" in operands else set()
    for first, last, single in re.findall(r"\bs\[(\d+):(\d+)\]|\bs(\d+)\b", operands):
        out |= {int(single)} if single else set(range(int(first), int(last) + 1))
    return out


def written_by_vector(op: str, operands: list):
    """The scalar registers that a vector instruction writes."""
    if op.startswith(("v_readfirstlane", "v_readlane")) or (op.startswith("v_cmp") and not op.startswith("v_cmpx")):
        return scalar_registers(operands[0])
    if ("_co_" in op or op.startswith(("v_mad_u64", "v_mad_i64", "v_div_scale"))) and len(operands) > 1:
        return scalar_registers(operands[1])
    return set()


def early_reads(lines):
    """Loads and stores that read a scalar register fewer than five wait states after a vector instruction wrote it: the
    hardware does not wait for it.  Instructions are taken in the order they stand in, a jump as one of them."""
    found, recent, kernel = [], [], ""
    for line in lines:
        line = line.split("//")[0].strip()
        if line.endswith(">:"):
            kernel, recent = line, []
            continue
        op, _, rest = line.partition(" ")
        if not op:
            continue
        operands = [o.strip() for o in rest.split(",")]
        if recent and op.startswith(("global_", "buffer_", "flat_", "scratch_")):
            read = scalar_registers(rest)
            found += [f"{kernel} {written} ... {line}" for age, registers, written in recent if age < 5 and registers & read]
        step = int(rest, 0) + 1 if op == "s_nop" else 1
        recent = [(age + step, registers, written) for age, registers, written in recent if age + step < 5]
        registers = written_by_vector(op, operands) if op.startswith("v_") else set()
        if registers:
            recent.append((0, registers, line))
    return found


def test_the_reader_of_device_code_sees_an_early_read():
    load = "global_load_lds_dwordx4 v6, s[4:5] nt"
    for between, early in ((["s_cbranch_scc0 12", "s_add_u32 m0, s19, 0", "s_nop 0"], True), (["s_nop 3"], True), (["s_nop 4"], False),
                           (["s_add_u32 m0, s19, 0", "s_nop 3"], False)):
        assert bool(early_reads(["<kernel>:", "v_readfirstlane_b32 s5, v18", *between, load])) == early
    assert early_reads(["v_readlane_b32 s4, v1, 3", load]) and early_reads(["v_cmp_gt_u32_e64 s[4:5], s0, v0", load])
    assert not early_reads(["v_readfirstlane_b32 s6, v18", load]) and not early_reads(["s_mov_b32 s4, s5", load])


@pytest.fixture(scope="module")
def device_code(tmp_path_factory):
    """The lines of every code object of the built library."""
    if not Path(OBJDUMP).exists():
        pytest.skip("no llvm-objdump here")
    out = []
    for code in code_objects(build.LIB_PATH.read_bytes()):
        path = tmp_path_factory.mktemp("code") / "object.co"
        path.write_bytes(code)
        out.append(subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", str(path)], check=True,
                                  stdout=subprocess.PIPE, text=True).stdout.splitlines())
    assert len(out) >= 10  # one for every file with kernels
    return out


def test_no_load_reads_a_scalar_register_that_is_still_being_written(device_code):
    found = [f for lines in device_code for f in early_reads(lines)]
    assert not found, f"{len(found)} loads, the first: {found[0]}"


def other_uses_of_m0(lines):
    """Instructions with M0 other than a load to LDS (which reads its address there) and, one wait state before it, the write
    that belongs to it."""
    code = [line.split("//")[0].strip() for line in lines]
    code = [line for line in code if line]
    found, mine = [], set()
    for i, line in enumerate(code):
        if line.startswith("global_load_lds_"):
            mine.add(i - 2)
            if not (re.match(r"s_(mov_b32|add_u32) m0, ", code[i - 2]) and code[i - 1].startswith("s_nop ")):
                found.append(line)
    for i, line in enumerate(code):
        if i not in mine and (re.search(r"\bm0\b", line) or re.match(r"v_movrel|s_movrel|s_set_gpr_idx|v_interp|s_sendmsg|ds_gws", line)):
            found.append(line)
    return found


def test_the_reader_of_device_code_sees_a_second_user_of_m0():
    own = ["s_add_u32 m0, s8, 0x400", "s_nop 0", "global_load_lds_dwordx4 v4, s[4:5] nt"]
    assert not other_uses_of_m0([*own, "s_add_u32 s8, s8, 1", *own])
    for line in ("s_mov_b32 m0, s3", "v_movrels_b32_e32 v1, v2", "s_set_gpr_idx_on s3, gpr_idx(SRC0)", "v_readlane_b32 s3, v1, m0"):
        assert other_uses_of_m0([*own, line, *own])
    assert other_uses_of_m0(own[1:]) and other_uses_of_m0([own[0], own[2]])


def test_nothing_but_the_loads_to_lds_uses_m0(device_code):
    """The statements that load to LDS write M0 and cannot say so (the compiler reserves the register and warns of it in a list
    of clobbers): nothing else may rely on what it holds."""
    found = [f for lines in device_code for f in other_uses_of_m0(lines)]
    assert not found, f"{len(found)} instructions, the first: {found[0]}"
    assert sum(line.lstrip().startswith("global_load_lds_") for lines in device_code for line in lines) > 1000

"""Wait states around the loads that write LDS, in the built library's own code.

These loads are issued from inline assembly, where the compiler does not see
what it would otherwise keep apart. gfx950 asks for one wait state between a
scalar write of m0 and a load that takes its LDS address from it, and for five
between a vector instruction's write of a scalar register and a load that reads
it. An instruction is one wait state, s_nop n is n + 1.
"""

from __future__ import annotations

import re
import shutil
import struct
import subprocess
from pathlib import Path

import pytest

from ssalaad_amd import library_path

MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def _objdump():
    at = Path("/opt/rocm/llvm/bin/llvm-objdump")
    return str(at) if at.exists() else shutil.which("llvm-objdump")


def _code_objects(data: bytes):
    at = -1
    while (at := data.find(MAGIC, at + 1)) >= 0:
        (count,) = struct.unpack_from("<Q", data, at + len(MAGIC))
        if count > 16:  # the name in some other place
            continue
        entry = at + len(MAGIC) + 8
        for _ in range(count):
            offset, size, name = struct.unpack_from("<QQQ", data, entry)
            target = data[entry + 24: entry + 24 + name]
            entry += 24 + name
            if target.endswith(b"gfx950"):
                yield data[at + offset: at + offset + size]


def _scalars(operand: str) -> set:
    if operand == "m0":
        return {"m0"}
    m = re.fullmatch(r"s\[(\d+):(\d+)\]|s(\d+)", operand)
    if not m:
        return set()
    return {int(m[3])} if m[3] else set(range(int(m[1]), int(m[2]) + 1))


def too_close(lines) -> list:
    """(instruction, the write it follows too closely) of every load into LDS."""
    bad, before = [], []
    for line in lines:
        words = re.split(r"[\s,]+", line.split("//")[0].strip())
        if len(words) < 2 or words[0].endswith(":"):
            continue
        if words[-1] == "lds":
            reads = set().union(*map(_scalars, words[1:]))
            states = 0
            for op, args in reversed(before[-5:]):
                if states >= 5:
                    break
                wrote = _scalars(args[0])
                if op.startswith("s_") and "m0" in wrote and states < 1:
                    bad.append((line.strip(), " ".join((op, *args))))
                if op.startswith("v_") and wrote & (reads | {"m0"}):
                    bad.append((line.strip(), " ".join((op, *args))))
                states += int(args[0], 0) + 1 if op == "s_nop" else 1
        before.append((words[0], words[1:]))
    return bad


def test_the_rules_on_short_listings():
    load = "buffer_load_dwordx4 v1, s[4:7], 0 offen lds"
    assert too_close(["s_mov_b32 m0, s8", load])
    assert not too_close(["s_mov_b32 m0, s8", "s_nop 0", load])
    assert too_close(["v_readlane_b32 s6, v1, s2", "s_mov_b32 m0, s8", "s_nop 2", load])
    assert not too_close(["v_readlane_b32 s6, v1, s2", "s_mov_b32 m0, s8", "s_nop 3", load])
    assert not too_close(["v_readlane_b32 s8, v1, s2", "s_mov_b32 m0, s8", "s_nop 0", load])


def test_loads_into_lds_wait_for_their_registers(tmp_path):
    tool = _objdump()
    if tool is None:
        pytest.skip("no llvm-objdump")
    loads = 0
    for code in _code_objects(Path(library_path()).read_bytes()):
        (tmp_path / "code").write_bytes(code)
        lines = subprocess.run([tool, "-d", "--no-show-raw-insn", "--no-leading-addr",
                                str(tmp_path / "code")], capture_output=True, text=True,
                               check=True).stdout.splitlines()
        mine = sum(line.split("//")[0].rstrip().endswith(" lds") for line in lines)
        loads += mine
        if mine:
            bad = too_close(lines)
            assert not bad, (len(bad), bad[0])
    assert loads  # the prefill's and the prompt attention's

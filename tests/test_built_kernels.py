"""CPU: what the built library's machine code has to hold.

A wave's reads of LDS return some time after they are issued, and s_barrier does
not wait for them.  Where a kernel reuses the memory behind a barrier, every
wave's reads have to have returned before it arrives there: an s_waitcnt
lgkmcnt(0) between the last read and the barrier on every path.  Results do not
show a missing one reliably, so the instructions are followed here."""
from __future__ import annotations

import os
import re
import shutil
import struct
import subprocess

import pytest

from tests.conftest import ROOT

LIB = os.path.join(ROOT, "see-ai_amd", "libseeai_hip.so")
OBJDUMP = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"


def code_objects(data):
    """The gfx950 code objects bundled in a library of this repository's own build."""
    magic, at = b"__CLANG_OFFLOAD_BUNDLE__", 0
    while (at := data.find(magic, at)) >= 0:
        count, = struct.unpack_from("<Q", data, at + len(magic))
        p = at + len(magic) + 8
        for _ in range(count):
            off, size, name = struct.unpack_from("<QQQ", data, p)
            p += 24
            if b"amdgcn" in data[p:p + name] and size:
                yield data[at + off:at + off + size]
            p += name
        at = p


def kernels(tmp_path, name):
    """(symbol, [(address, instruction, branch target or None)]) of the kernels whose symbol holds `name`."""
    with open(LIB, "rb") as f:
        data = f.read()
    for blob in code_objects(data):
        if name.encode() not in blob:
            continue
        path = tmp_path / "code.co"
        path.write_bytes(blob)
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(path)], check=True,
                              capture_output=True, text=True).stdout
        for part in re.split(r"\n(?=[0-9a-f]+ <)", text):
            head = re.match(r"([0-9a-f]+) <(.+)>:\n", part)
            if not head or name not in head[2]:
                continue
            start, code = int(head[1], 16), []
            for line in part.splitlines()[1:]:
                m = re.match(r"\s+(\S.*?)\s*// ([0-9A-F]+):", line)
                if m:
                    to = re.search(r"<.+\+0x([0-9a-f]+)>\s*$", line)
                    code.append((int(m[2], 16), m[1], start + int(to[1], 16) if to else None))
            yield head[2], code


def barriers_with_reads_in_flight(code):
    """Addresses of the s_barriers that a path reaches with a read of LDS not waited for."""
    index = {a: i for i, (a, _, _) in enumerate(code)}
    reached = [set() for _ in code]  # whether reads are in flight on arrival
    todo, found = [(0, False)], set()
    while todo:
        i, flying = todo.pop()
        while i < len(code) and flying not in reached[i]:
            reached[i].add(flying)
            address, text, target = code[i]
            op = text.split()[0]
            if op.startswith("ds_read"):
                flying = True
            elif op == "s_waitcnt" and ("lgkmcnt(0)" in text or text.split()[1:] == ["0"]):
                flying = False
            elif op == "s_barrier" and flying:
                found.add(address)
            if target is not None:
                todo.append((index[target], flying))
            assert not op.startswith(("s_setpc", "s_swappc")), "a jump that cannot be followed"
            if op in ("s_branch", "s_endpgm"):
                break
            i += 1
    return found


def test_the_walk_sees_a_missing_wait():
    def ask(*text, to=None):
        return barriers_with_reads_in_flight([(i, t, (to or {}).get(i)) for i, t in enumerate(text)])
    read, wait, end = "ds_read_b128 v[0:3], v4", "s_waitcnt vmcnt(0) lgkmcnt(0)", "s_endpgm"
    assert ask(read, wait, "s_barrier", end) == set()
    assert ask(read, "s_waitcnt vmcnt(0)", "s_barrier", end) == {2}
    assert ask(read, "s_waitcnt lgkmcnt(2)", "s_barrier", end) == {2}
    # round a loop, and past a branch that skips the wait
    assert ask("s_barrier", read, "s_cbranch_scc1 0", end, to={2: 0}) == {0}
    assert ask(read, "s_cbranch_scc0 2", wait, "s_barrier", end, to={1: 3}) == {3}


def test_feed_forward_tiles_wait_for_their_lds_reads_before_every_barrier(hip, tmp_path):
    """FfnMma's barriers all stand before memory that is written again: a stage's next loads, or
    the epilogue's staging over the last stage."""
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    seen, bad = 0, {}
    for name, code in kernels(tmp_path, "FfnMma"):
        seen += 1
        assert sum(text.startswith("s_barrier") for _, text, _ in code) >= 3, name
        if at := barriers_with_reads_in_flight(code):
            bad[name] = sorted(hex(a) for a in at)
    assert seen >= 20
    assert not bad, f"{len(bad)} of {seen}: {bad}"

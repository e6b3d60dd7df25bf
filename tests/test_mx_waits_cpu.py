"""The tile kernels' counted waits in the built library, from its assembly (no GPU).

With three and four buffers of x a step ends in a wait that leaves (kBufs - 2) steps' loads in flight: the tile that comes
next has arrived if those steps did issue as many.  The compiler drops loads whose result nobody reads, so the count is
checked where it stands, in the instructions."""

from __future__ import annotations

import os
import re
import struct
import subprocess

import pytest

from lastkv_amd import _lib

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


def code_objects(path):
    """The gfx950 code objects of a library (offload bundles: magic, count, then (offset, size, id length, id) each)."""

    data = path.read_bytes()
    for m in re.finditer(rb"__CLANG_OFFLOAD_BUNDLE__", data):
        (count,), at = struct.unpack_from("<Q", data, m.start() + 24), m.start() + 32
        for _ in range(count):
            offset, size, length = struct.unpack_from("<QQQ", data, at)
            name = data[at + 24:at + 24 + length]
            at += 24 + length
            if name.endswith(b"gfx950"):
                yield data[m.start() + offset:m.start() + offset + size]


def tile_kernels(tmp_path):
    """{(template arguments): its instructions} of mx4_tile_kernel."""

    _lib.load()
    found = {}
    for blob in code_objects(_lib.LIB_PATH):
        if b"mx4_tile_kernel" not in blob:
            continue
        (tmp_path / "code").write_bytes(blob)
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", str(tmp_path / "code")], check=True,
                              capture_output=True, text=True).stdout
        now = None
        for line in text.splitlines():
            m = re.match(r"<(\S+)>:", line)
            if m:
                args = re.search(r"mx4_tile_kernelILb(\d)" + r"ELi(\d+)" * 5, m.group(1))
                now = found.setdefault(tuple(int(v) for v in args.groups()), []) if args else None
            elif now is not None and line.strip():
                now.append(line.strip())
    return found


def overdrawn(lines, bufs):
    """Counted waits before a barrier that leave more loads in flight than the last bufs - 2 steps issued."""

    issued, counted, bad, wait = [0], 0, [], None
    for line in lines:
        op = line.split()[0]
        if op.startswith(("buffer_load", "global_load")):
            issued[-1] += 1
            wait = None
        elif op == "s_waitcnt" and "vmcnt" in line:
            wait = int(re.search(r"vmcnt\((\d+)\)", line).group(1))
        elif op == "s_barrier":
            if wait:
                counted += 1
                if wait > sum(issued[-(bufs - 2):] if bufs > 2 else []):
                    bad.append((len(issued), wait, issued[-4:]))
            issued.append(0)
            wait = None
    return counted, bad


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="needs the ROCm toolchain")
def test_waits_leave_no_more_than_the_steps_issued(tmp_path):
    kernels = tile_kernels(tmp_path)
    assert len(kernels) >= 5
    for args, lines in kernels.items():
        counted, bad = overdrawn(lines, args[-1])
        assert not bad, (args, bad)
        assert (counted >= 4) == (args[-1] > 2), (args, counted)  # (a unit's four steps)


def test_the_check_sees_an_overdrawn_wait():
    step = ["buffer_load_dword v0 lds"] * 4 + ["s_waitcnt vmcnt(%d)", "s_barrier"]
    fill = lambda n: [line % n if "%d" in line else line for line in step]
    assert overdrawn(fill(4) + fill(4), 3) == (2, [])
    assert overdrawn(fill(4) + fill(6), 3)[1] == [(2, 6, [4, 4])]
    assert overdrawn(fill(0) + fill(8), 4) == (1, [])

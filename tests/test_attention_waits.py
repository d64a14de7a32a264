"""The attention kernels' rescaling of their accumulators is inline assembly,
before which the compiler does not put the wait states that a matrix
instruction's result needs: every kernel has them itself.  Read in the
disassembly of the library that was built here."""
from __future__ import annotations

import re
import struct
import subprocess
from pathlib import Path

import pytest

from qwowl35_amd import build

OBJDUMP = Path("/opt/rocm/llvm/bin/llvm-objdump")


def _code_objects(blob: bytes):
    magic = b"__CLANG_OFFLOAD_BUNDLE__"
    at = blob.find(magic)
    while at >= 0:
        pos = at + len(magic) + 8
        for _ in range(struct.unpack_from("<Q", blob, pos - 8)[0]):
            offset, size, name_len = struct.unpack_from("<QQQ", blob, pos)
            pos += 24 + name_len
            elf = blob[at + offset:at + offset + size]
            if elf[:4] == b"\x7fELF":
                yield elf
        at = blob.find(magic, pos)


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """Instructions of each attention kernel, one a line."""
    if not OBJDUMP.exists():
        pytest.skip("no llvm-objdump")
    path, out = tmp_path_factory.mktemp("elf") / "code", {}
    for elf in _code_objects(build.LIB.read_bytes()):
        if b"prefix_attention_kernel" in elf:
            path.write_bytes(elf)
            text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", str(path)], check=True,
                                  capture_output=True, text=True).stdout
            for name, body in re.findall(r"<(\w*prefix_attention_kernel\w*)>:\n(.*?)(?=\n\n|\Z)", text, re.S):
                out[name] = [re.sub(r"\s*//.*", "", line).strip() for line in body.splitlines()]
    return out


def test_every_rescaling_waits(kernels):
    assert len(kernels) == 24
    for name, lines in kernels.items():
        waits = [i for i, line in enumerate(lines) if line == "s_nop 15" and lines[i + 1] == "s_nop 3"]
        assert waits, name
        # Accumulation registers are read, scaled and written back in three instructions: every such triple comes
        # after a wait, with no matrix instruction between them.
        scaled, ready = 0, False
        for i, line in enumerate(lines):
            if i in waits:
                ready = True
            elif line.startswith("v_mfma"):
                ready = False
            elif line.startswith("v_accvgpr_read_b32"):
                v, a = re.findall(r"[va]\d+", line)
                scale = lines[i + 1].startswith("v_mul_f32") and lines[i + 1].endswith(v)
                if scale and lines[i + 2] == f"v_accvgpr_write_b32 {a}, {v}":
                    scaled += 1
                    assert ready, (name, line)
        assert bool(scaled) == ("ILi256E" in name), name

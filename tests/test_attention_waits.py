"""The attention kernels rescale their accumulators by inline assembly, before
which the compiler does not put the wait states that a matrix instruction's
result needs: here they are counted, along every path, in the disassembly of the
library that was built here."""
from __future__ import annotations

import re
import struct
import subprocess
from pathlib import Path

import pytest

from qwowl35_amd import build

OBJDUMP = Path("/opt/rocm/llvm/bin/llvm-objdump")
# wait states from a matrix instruction to an access of its result: of 8 passes, of 4
NEEDS = {"v_mfma_f32_32x32x16": 12, "v_mfma_f32_16x16x32": 8}


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


def _registers(text: str) -> set:
    out = set()
    for kind, one, lo, hi in re.findall(r"\b([va])(?:(\d+)\b|\[(\d+):(\d+)\])", text):
        out |= {kind + one} if one else {kind + str(i) for i in range(int(lo), int(hi) + 1)}
    return out


def _disassembly(elf: bytes, path: Path):
    """(name, [(address, instruction, branch target or None)]) of each attention kernel."""
    path.write_bytes(elf)
    text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(path)], check=True, capture_output=True,
                          text=True).stdout
    for start, name, body in re.findall(r"^([0-9a-f]+) <(\w*prefix_attention_kernel\w*)>:\n(.*?)(?=^\n|\Z)", text, re.S | re.M):
        code = []
        for line in body.splitlines():
            m = re.match(r"\s+(\S.*?)\s*//\s*([0-9A-F]+):", line)
            if m:
                target = re.search(r"<\w+\+0x([0-9a-f]+)>", line)
                code.append((int(m.group(2), 16), m.group(1), int(start, 16) + int(target.group(1), 16) if target else None))
        yield name, code


def _too_early(code) -> list:
    """Accesses of a matrix instruction's result by others before it is there."""
    index = {at: i for i, (at, _, _) in enumerate(code)}
    ops = []
    for at, text, target in code:
        op = text.split()[0]
        need = next((n for k, n in NEEDS.items() if op.startswith(k)), 0)
        assert need or "mfma" not in op, text
        regs = _registers(text.split(",")[0]) if need else _registers(text) if op[:2] in ("v_", "ds", "gl", "bu", "fl") else set()
        steps = int(text.split()[1], 0) + 1 if op == "s_nop" else 1
        follow = []
        if op not in ("s_branch", "s_endpgm", "s_setpc_b64"):
            follow.append(index[at] + 1)
        if op.startswith(("s_branch", "s_cbranch")):
            follow.append(index[target])
        ops.append((op, need, regs, steps, follow))
    pending = [None] * len(ops)  # at each instruction: register -> wait states it still needs
    pending[0], work, bad = {}, [0], {}
    while work:
        i = work.pop()
        op, need, regs, steps, follow = ops[i]
        state = pending[i]
        if not need:
            for r in regs & state.keys():
                bad[i] = (code[i], r, state[r])
        after = {r: n - steps for r, n in state.items() if n > steps}
        if need:
            after |= dict.fromkeys(regs, need)
        for j in follow:
            if j >= len(ops):
                continue
            if pending[j] is None:
                pending[j] = dict(after)
            elif any(pending[j].get(r, 0) < n for r, n in after.items()):
                for r, n in after.items():
                    pending[j][r] = max(pending[j].get(r, 0), n)
            else:
                continue
            work.append(j)
    return list(bad.values())


def test_every_access_of_a_product_waits_for_it(tmp_path):
    if not OBJDUMP.exists():
        pytest.skip("no llvm-objdump")
    seen, rescaled = 0, 0
    for elf in _code_objects(build.LIB.read_bytes()):
        if b"prefix_attention_kernel" not in elf:
            continue
        for name, code in _disassembly(elf, tmp_path / "code"):
            seen += 1
            early = _too_early(code)
            assert not early, (name, early[:5])
            rescaled += any(a[1].startswith("v_accvgpr_read") and b[1].startswith("v_mul_f32")
                            and c[1].startswith("v_accvgpr_write") for a, b, c in zip(code, code[1:], code[2:]))
    assert seen == 24 and rescaled == 8  # (256 columns: in accumulation registers)


def test_the_count_finds_an_early_access():
    """The counting itself, on a few instructions, over a branch."""
    mfma = "v_mfma_f32_32x32x16_f16 a[0:15], v[0:3], v[4:7], a[0:15]"
    code = [(0, mfma, None), (8, "s_cbranch_vccz 3", 40), (16, "s_nop 9", None), (24, "v_accvgpr_read_b32 v9, a3", None),
            (32, "s_endpgm", None), (40, "s_nop 15", None), (48, "v_accvgpr_read_b32 v9, a15", None), (56, "s_endpgm", None)]
    assert [b[1:] for b in _too_early(code)] == [("a3", 1)]
    code[2] = (16, "s_nop 10", None)
    assert not _too_early(code)

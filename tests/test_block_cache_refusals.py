"""Argument checks of the block-scaled cache's calls, which need no GPU, and what the compiler made of their kernels."""
from __future__ import annotations

import ctypes as C
import re
import subprocess

import pytest

from qwowl35_amd import _ffi, build
from qwowl35_amd._ffi import Qw35Error
from tests.test_attention_refusals import AT, HEADER, attend, cache, heads
from tests.test_attention_waits import OBJDUMP, _code_objects, _too_early
from tests.test_kernel_resources import _kernels

BLOCKS = [_ffi.DTYPE_E4M3_BLOCKS, _ffi.DTYPE_I8_BLOCKS]


def blocks(dtype=_ffi.DTYPE_I8_BLOCKS, **kw):
    return cache(**{"dtype": dtype, "k_scale": AT, "v_scale": AT, **kw})


def read(c=None, k=None, v=None, n=2, slots=AT):
    return _ffi.call("qw35_hip_kv_read", C.byref(c or blocks()), C.byref(k or heads()), C.byref(v or heads()), n, slots, None)


def append(c, n=1, k=None, v=None, slots=AT):
    return _ffi.call("qw35_hip_kv_append", C.byref(c), C.byref(k or heads()), C.byref(v or heads()), n, slots, None, None, 0,
                     None, 0.0, None)


def test_types_match_the_header():
    text = HEADER.read_text()
    for name, value in (("E4M3_BLOCKS", _ffi.DTYPE_E4M3_BLOCKS), ("I8_BLOCKS", _ffi.DTYPE_I8_BLOCKS)):
        assert re.search(rf"#define QW35_HIP_DTYPE_{name} {value}u", text)


@pytest.mark.parametrize("dtype", BLOCKS)
@pytest.mark.parametrize("message,kw", [
    ("null cache", {"v": None}),
    ("null scales", {"k_scale": None}),
    ("null scales", {"v_scale": None}),
    ("their scales 4-byte", {"v_scale": AT + 2}),
    ("16-byte aligned", {"k": AT + 8}),
    ("head_dim=96", {"head_dim": 96}),
    ("page_size=48", {"page_size": 48}),
    ("kv_heads=0", {"kv_heads": 0}),
    ("2^32 - 2 blocks", {"n_pages": 1 << 30, "page_size": 128}),
])
def test_caches_refused(dtype, message, kw):
    c = blocks(dtype, **kw)
    for call in (append, read, lambda c: attend(c=c)):
        with pytest.raises(Qw35Error, match=re.escape(message)):
            call(c)
    assert _ffi.load().qw35_hip_prefix_attention_workspace_size(C.byref(c), 4, 1, 1) == 0


@pytest.mark.parametrize("message,kw", [
    ("null k", {"k": heads(data=None)}),
    ("null v", {"v": heads(data=None)}),
    ("k must be f32, bf16 or f16", {"k": heads(_ffi.DTYPE_I8_BLOCKS)}),
    ("one type", {"k": heads(_ffi.DTYPE_F16)}),
    ("aligned to its elements", {"v": heads(data=AT + 2)}),
    ("n_tokens=", {"n": 1 << 23}),
    ("slots", {"slots": None}),
    ("slots", {"slots": AT + 4}),
])
@pytest.mark.parametrize("c", [None, cache()])
def test_read_refuses(message, kw, c):
    with pytest.raises(Qw35Error, match=re.escape(message)):
        read(c, **kw)


def test_nothing_to_do_is_done():
    assert read(n=0) == 1 and append(blocks(), n=0) == 1


def test_query_types():
    for dtype, q, fine in ((_ffi.DTYPE_I8_BLOCKS, _ffi.DTYPE_BF16, False), (_ffi.DTYPE_I8_BLOCKS, _ffi.DTYPE_F32, False),
                           (_ffi.DTYPE_E4M3_BLOCKS, _ffi.DTYPE_F32, False), (_ffi.DTYPE_I8_BLOCKS, _ffi.DTYPE_F16, True),
                           (_ffi.DTYPE_E4M3_BLOCKS, _ffi.DTYPE_F16, True), (_ffi.DTYPE_E4M3_BLOCKS, _ffi.DTYPE_BF16, True)):
        with pytest.raises(Qw35Error, match="workspace" if fine else "q must have the cache's type"):
            attend(c=blocks(dtype), q=heads(q), workspace=None)


@pytest.mark.parametrize("dtype", BLOCKS)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_the_workspace_is_a_16_bit_caches_or_none(dim, dtype):
    """Scales beside the marks take room from the list of row tiles: larger batches than that has are refused, by size
    and call."""
    lib = _ffi.load()
    like, mine = cache(head_dim=dim), blocks(dtype, head_dim=dim)
    size = lambda c, n: lib.qw35_hip_prefix_attention_workspace_size(C.byref(c), 2, n, n)  # noqa: E731
    assert size(mine, 8) == size(like, 8)
    last = max(n for n in range(1000, 9000) if size(mine, n))
    assert size(mine, last + 1) == 0 and bool(size(like, last + 1)) == (dtype == _ffi.DTYPE_E4M3_BLOCKS)
    with pytest.raises(Qw35Error, match="row tiles in a call"):
        attend(c=mine, n_heads=2, n_seqs=last + 1, n_tokens=last + 1)
    with pytest.raises(Qw35Error, match="needs a 256-byte aligned workspace"):
        attend(c=mine, n_heads=2, n_seqs=last, n_tokens=last, workspace=None)


def test_kernels_keep_their_registers():
    kernels = [k for k in _kernels(build.LIB.read_bytes())
               if any(n in k[".name"] for n in ("block_attention_kernel", "append_blocks", "kv_read"))]
    main = [k for k in kernels if "block_attention_kernel" in k[".name"]]
    assert len(main) == 18  # three head sizes, three pairs of queries and codes, with and without shared tiles
    spilled = {k[".name"]: k[".vgpr_spill_count"] for k in kernels if k[".vgpr_spill_count"]}
    assert not spilled, spilled
    for k in main:  # one wave a SIMD of 256 columns, two of less
        assert k[".vgpr_count"] <= (512 if "ILi256E" in k[".name"] else 256), k[".name"]


def _kernel_code(elf: bytes, path):
    """(name, [(address, instruction, branch target or None)]) of each kernel over a block-scaled cache."""
    path.write_bytes(elf)
    text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(path)], check=True, capture_output=True, text=True).stdout
    for start, name, body in re.findall(r"^([0-9a-f]+) <(\w*block_attention_kernel\w*)>:\n(.*?)(?=^\n|\Z)", text, re.S | re.M):
        lines = [m for m in (re.match(r"\s+(\S.*?)\s*//\s*([0-9A-F]+):(.*)", line) for line in body.splitlines()) if m]
        targets = [re.search(r"<\w+\+0x([0-9a-f]+)>", m.group(0)) for m in lines]
        yield name, [(int(m.group(2), 16), m.group(1), int(start, 16) + int(t.group(1), 16) if t else None)
                     for m, t in zip(lines, targets)]


def test_every_access_of_a_product_waits_for_it(tmp_path):
    """As for the other caches' kernels: wait states before the rescaling's inline assembly, counted in the library."""
    if not OBJDUMP.exists():
        pytest.skip("no llvm-objdump")
    seen = 0
    for elf in _code_objects(build.LIB.read_bytes()):
        if b"block_attention_kernel" not in elf:
            continue
        for name, code in _kernel_code(elf, tmp_path / "code"):
            seen += 1
            early = _too_early(code)
            assert not early, (name, early[:5])
    assert seen == 18

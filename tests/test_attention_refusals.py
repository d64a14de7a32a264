"""The attention entry points' argument checks, which need no GPU: every call below ends before any device work."""
from __future__ import annotations

import ctypes as C
import re
import subprocess
from pathlib import Path

import pytest

from qwowl35_amd import _ffi
from qwowl35_amd._ffi import Qw35Error

HEADER = Path(__file__).resolve().parents[1] / "include" / "qw35_hip.h"
AT = 4096  # a stand-in device address


def heads(dtype=_ffi.DTYPE_F32, data=AT, token=512, head=64):
    return _ffi.Heads(data, token, head, dtype, 0)


def rope(rot=32, sections=(), interleaved=0, freq=AT):
    return _ffi.Rope(freq, rot, interleaved, (C.c_uint32 * 4)(*(list(sections) + [0] * (4 - len(sections)))))


def cache(**kw):
    c = _ffi.KvCache(AT, AT, None, None, 8, 64, 2, 64, _ffi.DTYPE_F16, 0)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def test_struct_layouts_match_the_header(tmp_path):
    names = {"heads": _ffi.Heads, "rope": _ffi.Rope, "kv_cache": _ffi.KvCache, "attention": _ffi.Attention}
    lines, want = [], []
    for name, mirror in names.items():
        lines.append(f'printf("%zu\\n", sizeof(qw35_hip_{name}));')
        want.append(C.sizeof(mirror))
        for field, *_ in mirror._fields_:
            lines.append(f'printf("%zu\\n", offsetof(qw35_hip_{name}, {field}));')
            want.append(getattr(mirror, field).offset)
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "qw35_hip.h"\nint main(void){\n'
                   + "\n".join(lines) + "\nreturn 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-I", str(HEADER.parent), str(src), "-o", str(exe)], check=True)
    got = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()
    assert [int(v) for v in got] == want
    text = HEADER.read_text()
    for name, value in (("F16", _ffi.DTYPE_F16), ("E4M3", _ffi.DTYPE_E4M3)):
        assert re.search(rf"#define QW35_HIP_DTYPE_{name} {value}u", text)


def rotate(x=None, y=None, n=2, h=2, dim=64, r=None, pos=AT, axes=1, norm=None, eps=1e-6):
    x = x or heads()
    y = y or heads()
    return _ffi.call("qw35_hip_rotate", C.byref(x), C.byref(y), n, h, dim, C.byref(r) if r else None, pos, axes, norm,
                     eps, None)


@pytest.mark.parametrize("message,kw", [
    ("dim=60 must be a multiple of 8", {"dim": 60}),
    ("dim=520", {"dim": 520}),
    ("heads=0", {"h": 0}),
    ("n_tokens=8388608", {"n": 1 << 23}),
    ("null x", {"x": heads(data=None)}),
    ("null y", {"y": heads(data=None)}),
    ("x must be f32, bf16 or f16", {"x": heads(_ffi.DTYPE_E4M3)}),
    ("aligned to its elements", {"x": heads(data=AT + 2)}),
    ("rot_dim=24", {"r": rope(24)}),
    ("rot_dim=80", {"r": rope(80)}),
    ("rot_dim=0", {"r": rope(0)}),
    ("frequencies", {"r": rope(freq=None)}),
    ("add up to rot_dim / 2 = 16", {"r": rope(32, [5, 5, 5])}),
    ("does not fit 16 interleaved pairs", {"r": rope(32, [4, 6, 6], 1), "axes": 3}),
    ("three axes", {"r": rope(32, [4, 4, 4, 4], 1), "axes": 4}),
    ("positions have 2 axes, the sections 1 or 3", {"r": rope(32, [6, 5, 5]), "axes": 2}),
    ("positions must be", {"r": rope(), "pos": None}),
    ("norm must be 4-byte aligned", {"norm": AT + 1}),
    ("eps must be", {"norm": AT, "eps": -1.0}),
    ("eps must be", {"norm": AT, "eps": float("nan")}),
])
def test_rotate_refuses(message, kw):
    with pytest.raises(Qw35Error, match=re.escape(message)):
        rotate(**kw)


def test_nothing_to_do_is_done():
    assert rotate(n=0) == 1
    c = cache()
    assert _ffi.call("qw35_hip_kv_append", C.byref(c), C.byref(heads()), C.byref(heads()), 0, None, None, None, 0,
                     None, 0.0, None) == 1


CACHES = [
    ("null cache", {"k": None}),
    ("16-byte aligned", {"v": AT + 8}),
    ("a cache is f16, bf16 or e4m3", {"dtype": _ffi.DTYPE_F32}),
    ("only an e4m3 cache has scales", {"k_scale": AT}),
    ("head_dim=96", {"head_dim": 96}),
    ("page_size=48", {"page_size": 48}),
    ("page_size=0", {"page_size": 0}),
    ("kv_heads=0", {"kv_heads": 0}),
    ("n_pages=0", {"n_pages": 0}),
    ("2^32 - 2 blocks", {"n_pages": 1 << 30, "page_size": 128}),
]


@pytest.mark.parametrize("message,kw", CACHES)
def test_caches_refused(message, kw):
    c = cache(**kw)
    with pytest.raises(Qw35Error, match=re.escape(message)):
        _ffi.call("qw35_hip_kv_append", C.byref(c), C.byref(heads()), C.byref(heads()), 1, AT, None, None, 0, None,
                  0.0, None)
    with pytest.raises(Qw35Error, match=re.escape(message)):
        attend(c=c)
    assert _ffi.load().qw35_hip_prefix_attention_workspace_size(C.byref(c), 4, 1, 1) == 0


@pytest.mark.parametrize("message,args", [
    ("one type", {"v": heads(_ffi.DTYPE_BF16)}),
    ("slots", {"slots": None}),
    ("slots", {"slots": AT + 4}),
    ("null k", {"k": heads(data=None)}),
    ("null v", {"v": heads(data=None)}),
    ("n_tokens=", {"n": 1 << 23}),
    ("rot_dim=80", {"r": rope(80)}),
])
def test_kv_append_refuses(message, args):
    a = {"k": heads(), "v": heads(), "n": 2, "slots": AT, "r": None, **args}
    c = cache()
    with pytest.raises(Qw35Error, match=re.escape(message)):
        _ffi.call("qw35_hip_kv_append", C.byref(c), C.byref(a["k"]), C.byref(a["v"]), a["n"], a["slots"],
                  C.byref(a["r"]) if a["r"] else None, AT, 1, None, 0.0, None)


def attend(c=None, **kw):
    op = _ffi.Attention()
    op.q, op.out = heads(_ffi.DTYPE_F16), heads(_ffi.DTYPE_F16)
    op.n_tokens, op.n_heads, op.n_seqs = 2, 4, 2
    op.lengths = op.pages = AT
    op.pages_per_seq, op.scale = 4, 0.125
    op.workspace, op.workspace_bytes = AT, 1 << 40
    for k, v in kw.items():
        setattr(op, k, v)
    return _ffi.call("qw35_hip_prefix_attention", C.byref(op), C.byref(c or cache()), None)


@pytest.mark.parametrize("message,kw", [
    ("n_heads=3 must be a multiple of kv_heads=2", {"n_heads": 3}),
    ("n_heads=0", {"n_heads": 0}),
    ("n_tokens=", {"n_tokens": 1 << 23}),
    ("n_seqs=70000", {"n_seqs": 70000}),
    ("null q", {"q": heads(_ffi.DTYPE_F16, data=None)}),
    ("null out", {"out": heads(data=None)}),
    ("q must have the cache's type", {"q": heads(_ffi.DTYPE_BF16)}),
    ("q must have the cache's type", {"q": heads(_ffi.DTYPE_F32)}),
    ("out must be f32, bf16 or f16", {"out": heads(_ffi.DTYPE_E4M3)}),
    ("gate must be f32, bf16 or f16", {"gate": heads(7)}),
    ("without starts n_seqs=1 must be n_tokens=2", {"n_seqs": 1}),
    ("null lengths or pages", {"lengths": None}),
    ("null lengths or pages", {"pages": None}),
    ("4-byte aligned", {"starts": AT + 2}),
    ("2^30 positions", {"pages_per_seq": 1 << 25}),
    ("do not hold prefix_len=65", {"prefix_len": 65, "prefix_pages": AT, "n_prefix_pages": 1}),
    ("do not hold prefix_len=1", {"prefix_len": 1}),
    ("scale must be finite", {"scale": float("inf")}),
    ("scale must be finite", {"scale": float("nan")}),
    ("window=", {"window": (1 << 30) + 1}),
    ("sink=", {"sink": 0xffffffff}),
    ("row tiles in a call", {"n_tokens": 20000, "n_seqs": 20000}),
    ("workspace", {"workspace": None}),
    ("workspace", {"workspace": AT + 64}),
    ("workspace", {"workspace_bytes": 1024}),
])
def test_prefix_attention_refuses(message, kw):
    with pytest.raises(Qw35Error, match=re.escape(message)):
        attend(**kw)


def test_an_e4m3_cache_takes_either_query_type_but_no_fp32():
    with pytest.raises(Qw35Error, match="q must have the cache's type"):
        attend(c=cache(dtype=_ffi.DTYPE_E4M3), q=heads(_ffi.DTYPE_F32))
    with pytest.raises(Qw35Error, match="workspace"):  # (the check after it)
        attend(c=cache(dtype=_ffi.DTYPE_E4M3), q=heads(_ffi.DTYPE_BF16), workspace=None)


@pytest.mark.parametrize("seqs,tokens", [(1, 1), (8, 8), (64, 64), (3, 300), (1, 2048)])
def test_the_workspace_serves_every_division_of_the_rows(seqs, tokens):
    """Whatever max_new and prefix a call names, and for smaller batches too."""
    lib, c = _ffi.load(), cache(n_pages=1 << 16)
    for n_heads in (2, 4, 14, 64):
        size = lib.qw35_hip_prefix_attention_workspace_size(C.byref(c), n_heads, seqs, tokens)
        assert size
        for s, t in {(seqs, tokens), (max(1, seqs // 2), max(1, tokens // 2)), (1, max(1, tokens // 3))}:
            for new in {0, 1, 2, 3, 7, 16, 100, t}:
                for prefix in (0, 64):
                    if new <= t:
                        with pytest.raises(Qw35Error, match="needs a 256-byte aligned workspace of") as e:
                            attend(c=c, n_heads=n_heads, n_seqs=s, n_tokens=t, max_new=new, starts=AT,
                                   prefix_len=prefix, prefix_pages=AT, n_prefix_pages=1, workspace=None)
                        need = int(re.search(r"of (\d+) bytes", str(e.value)).group(1))
                        assert need <= size, (n_heads, s, t, new, prefix)


@pytest.mark.parametrize("rot,base", [(0, 1e4), (24, 1e4), (1024, 1e4), (32, 1.0), (32, float("inf")),
                                      (32, float("nan"))])
def test_rope_frequencies_refused(rot, base):
    out = (C.c_uint64 * 512)()
    with pytest.raises(Qw35Error, match="rope_freq"):
        _ffi.call("qw35_hip_rope_freq", rot, base, out)


def test_rope_frequencies():
    """Turns per position as 64-bit fractions, to the last few bits."""
    from fractions import Fraction

    out = (C.c_uint64 * 32)()
    _ffi.call("qw35_hip_rope_freq", 64, 16.0, out)  # 16^(-2 i / 64) = 2^(-i / 8): exact for i = 8 j
    two_pi = Fraction(6283185307179586476925286766559005768394, 10 ** 39)
    for j in range(4):
        exact = Fraction(2 ** 64, 2 ** j) / two_pi
        assert abs(out[8 * j] - exact) < 4, j


def test_python_checks_come_before_any_device_work():
    import torch

    from qwowl35_amd import attention as at

    x = torch.zeros(2, 3, 64)
    with pytest.raises(Qw35Error, match="device tensor"):
        at.rotate(x, None)
    with pytest.raises(Qw35Error, match="up to four counts"):
        at.Rotary(64, 1e4, [1, 2, 3, 4, 5], device="cpu")
    with pytest.raises(Qw35Error, match="rot_dim=64"):
        at.Rotary(64, 1e4, [10, 10, 10], device="cpu")
    with pytest.raises(Qw35Error, match="page_size=40"):
        at.PagedCache.empty(1, 1, 40, 64, device="cpu")
    with pytest.raises(Qw35Error, match="contiguous"):
        at.PagedCache(torch.zeros(1, 1, 1, 8, 32, 8), torch.zeros(1, 1, 4, 64, 8))


@pytest.mark.parametrize("n_heads,seqs,tokens", [(2, 200, 400), (4, 33, 2000), (16, 1000, 1000)])
def test_the_workspace_serves_fewer_sequences(n_heads, seqs, tokens):
    """Few sequences have their rows in larger units than many."""
    lib, c = _ffi.load(), cache(n_pages=1 << 16)
    size = lib.qw35_hip_prefix_attention_workspace_size(C.byref(c), n_heads, seqs, tokens)
    for s in (1, 15, 16, 31, 32, 33, 64, 65, seqs):
        for new in (1, 9, 20, 33, 64, 65, tokens):
            with pytest.raises(Qw35Error, match="needs a 256-byte aligned workspace of") as e:
                attend(c=c, n_heads=n_heads, n_seqs=min(s, seqs), n_tokens=tokens, max_new=new, starts=AT, workspace=None)
            assert int(re.search(r"of (\d+) bytes", str(e.value)).group(1)) <= size, (s, new)


@pytest.mark.parametrize("seqs", [1, 8, 64, 300])
@pytest.mark.parametrize("max_new", [0, 1, 7])
def test_a_token_each_is_divided_as_such(seqs, max_new):
    """Without starts max_new does not matter: rows are divided as for one new token of a sequence."""
    need = []
    c = cache(n_pages=1 << 16, kv_heads=4, head_dim=256)
    for kw in ({"max_new": max_new}, {"max_new": 1}):
        with pytest.raises(Qw35Error, match="needs a 256-byte aligned workspace of") as e:
            attend(c=c, n_heads=16, n_seqs=seqs, n_tokens=seqs, workspace=None, **kw)
        need.append(int(re.search(r"of (\d+) bytes", str(e.value)).group(1)))
    assert need[0] == need[1]


def _needs(c, heads, seqs, tokens, starts, max_new=0):
    """The workspace that a call asks for; 0: it has more row tiles than the list holds."""
    with pytest.raises(Qw35Error) as e:
        attend(c=c, n_heads=heads, n_seqs=seqs, n_tokens=tokens, starts=starts, max_new=max_new, workspace=None)
    m = re.search(r"workspace of (\d+) bytes", str(e.value))
    assert m or "row tiles in a call" in str(e.value), str(e.value)
    return int(m.group(1)) if m else 0


@pytest.mark.parametrize("dim,kv,heads", [(256, 4, 16), (256, 1, 16), (128, 2, 40), (64, 3, 3)])
def test_the_size_and_the_call_agree_on_what_is_too_much(dim, kv, heads):
    """On either side of the largest batch of single tokens, and of the largest chunk."""
    lib, c = _ffi.load(), cache(n_pages=1 << 16, kv_heads=kv, head_dim=dim)
    size = lambda s, t: lib.qw35_hip_prefix_attention_workspace_size(C.byref(c), heads, s, t)  # noqa: E731

    def largest(serves):
        lo, hi = 1, 1 << 22
        while lo < hi:
            mid = (lo + hi + 1) // 2
            lo, hi = (mid, hi) if serves(mid) else (lo, mid - 1)
        return lo

    most = largest(lambda n: n < 65536 and _needs(c, heads, n, n, None))
    room = {256: 1500, 128: 6000, 64: 6000}[dim]
    assert most >= room // (1 if heads // kv <= 16 else 2)
    for n in (most - 1, most):
        assert size(n, n) >= _needs(c, heads, n, n, None) > 0
    assert size(65535, 65535) == 0 and _needs(c, heads, 65535, 65535, None) == 0
    chunk = largest(lambda n: _needs(c, heads, 1, n, AT))
    assert size(1, chunk) >= _needs(c, heads, 1, chunk, AT) > 0
    assert size(1, chunk + 1) == 0
    # what a size serves, smaller batches have room in, however their rows are divided
    group = heads // kv
    for seqs, tokens in ((most, most), (most // 2, most), (1, chunk), (7, chunk // 3)):
        have = size(seqs, tokens)
        for s in {1, seqs // 3 + 1, seqs}:
            for t in {s, tokens // 2, tokens}:
                if not s <= t:
                    continue
                for new in {1, 16 // group or 1, 64 // group or 1, 64 // group + 1, t}:
                    assert _needs(c, heads, s, t, AT, min(new, t)) <= have
                if s == t:
                    assert _needs(c, heads, s, t, None) <= have

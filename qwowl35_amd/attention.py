"""Attention between the projections: rotary positions, a paged key/value cache
and attention of a batch that shares a prefix, over the C ABI.

An attention layer of the reference runs its q / k / v projections, one kernel
that norms, rotates and caches, flash attention and the output projection
(qw35-server/src/metal/bridge/Qw35MetalRuntime+Attention.m:35-113).  Here:

* ``rotate``            RMS norm and multi-axis rotary of the queries
* ``kv_append``         the same of the keys, and keys and values into the cache,
  which may hold them in 8 bits with a scale for each 32 tokens of a head
* ``kv_read``           tokens of a cache back as numbers
* ``prefix_attention``  softmax attention of one or more new tokens of each
  sequence over the shared prefix (read once for the batch) and their own pages

``GatedAttention`` runs a whole layer of them with the projections.

Device memory and streams come from torch; every computation is a call into
``libqw35_hip.so``, asynchronous on the current stream.  With another ``stream``
a call runs there, behind what the current one holds by then, and what it makes
is that stream's memory; to leave the current stream's work aside, call under
``torch.cuda.stream(stream)`` instead, with the inputs synchronised.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import math
import struct

import torch

from . import _ffi
from . import runtime as rt
from ._ffi import Qw35Error

_FLOAT = {torch.float32: _ffi.DTYPE_F32, torch.bfloat16: _ffi.DTYPE_BF16, torch.float16: _ffi.DTYPE_F16}
_CACHE = {torch.bfloat16: _ffi.DTYPE_BF16, torch.float16: _ffi.DTYPE_F16, torch.float8_e4m3fn: _ffi.DTYPE_E4M3}
_BLOCKS = {torch.float8_e4m3fn: _ffi.DTYPE_E4M3_BLOCKS, torch.int8: _ffi.DTYPE_I8_BLOCKS}

# A small call's time is this module's: structs are packed rather than built
# field by field, and their functions take addresses as plain numbers.
_HEADS = struct.Struct("=QqqII")
_ATTENTION = struct.Struct("=" + 3 * "QqqII" + "4I4Q5IfQQ")
_NO_HEADS = (0, 0, 0, 0, 0)
assert _HEADS.size == C.sizeof(_ffi.Heads) and _ATTENTION.size == C.sizeof(_ffi.Attention)
_at, _u32, _err = C.c_void_p, C.c_uint32, [C.c_char_p, C.c_size_t]
_ARGS = {
    "qw35_hip_rotate": [_at, _at, _u32, _u32, _u32, _at, _at, _u32, _at, C.c_float, _at],
    "qw35_hip_kv_append": [_at, _at, _at, _u32, _at, _at, _at, _u32, _at, C.c_float, _at],
    "qw35_hip_kv_read": [_at, _at, _at, _u32, _at, _at],
    "qw35_hip_prefix_attention": [_at, _at, _at],
}
_functions: dict = {}


def _call(name: str, *args) -> None:
    fn = _functions.get(name)
    if fn is None:
        fn = _functions[name] = C.CFUNCTYPE(C.c_int, *_ARGS[name], *_err)((name, _ffi.load()))
    err = _ffi._ErrBuffer()
    if not fn(*args, err, 512):
        raise Qw35Error(f"{name}: {err.value.decode(errors='replace')}")


def _elsewhere(device: int) -> bool:
    """Whether a call over tensors on cuda:``device`` has to make that device the current one first."""
    return device >= 0 and device != torch.cuda.current_device()


@contextlib.contextmanager
def _behind(stream, x: torch.Tensor):
    """``stream`` as the current one, behind what the one before holds."""
    if stream.device != x.device:
        raise Qw35Error(f"the stream is on {stream.device}, the input on {x.device}")
    stream.wait_stream(torch.cuda.current_stream(x.device))
    with torch.cuda.stream(stream):
        yield


def _heads(x: torch.Tensor, name: str) -> tuple:
    """The fields of the ``qw35_hip_heads`` of a [n_tokens, heads, dim] tensor with unit column stride."""
    code = _FLOAT.get(x.dtype)
    if code is None or not x.is_cuda or x.dim() != 3:
        raise Qw35Error(f"{name} must be an fp32, bf16 or fp16 [n_tokens, heads, dim] device tensor")
    token, head, column = x.stride()
    if column != 1 and x.shape[2] > 1:
        raise Qw35Error(f"{name} must have unit column stride, got strides {x.stride()}")
    return x.data_ptr(), token, head, code, 0


def _index(x: torch.Tensor, dtype: torch.dtype, shape: tuple, device: int, name: str) -> int:
    """The address of a contiguous tensor of that type and shape on cuda:``device``."""
    if x.dtype is not dtype or x.shape != shape or x.get_device() != device or not x.is_contiguous():
        raise Qw35Error(f"{name} must be a contiguous {dtype} {list(shape)} tensor on cuda:{device}, got "
                        f"{x.dtype} {list(x.shape)} on {x.device}")
    return x.data_ptr()


def _vector(x: torch.Tensor | None, n: int, device: int, name: str) -> int | None:
    return None if x is None else _index(x, torch.float32, (n,), device, name)


def _output(out: torch.Tensor | None, dtype: torch.dtype | None, like: torch.Tensor) -> torch.Tensor:
    """``out``, or a new tensor of like's shape."""
    if out is None:
        return torch.empty_like(like, dtype=dtype, memory_format=torch.contiguous_format)
    if out.shape != like.shape or out.device != like.device or (dtype or out.dtype) != out.dtype:
        raise Qw35Error(f"out must be a {list(like.shape)} tensor of out_dtype on {like.device}")
    return out


class Rotary:
    """Rotary positions: ``rot_dim`` columns (a multiple of 16) of a head turn by
    ``position * base^(-2 i / rot_dim)``, pair i being columns i and i + rot_dim / 2.

    ``sections`` gives the pairs of each axis (time, height, width, extra:
    ``rope_sections``), in a row or ``interleaved``; without it there is one axis."""

    def __init__(self, rot_dim: int, base: float, sections=None, interleaved: bool = False, device="cuda"):
        sections = [int(s) for s in (sections or [])]
        if len(sections) > 4 or any(s < 0 for s in sections):
            raise Qw35Error(f"rotary sections must be up to four counts, got {sections}")
        if rot_dim <= 0 or rot_dim % 16 or (sum(sections) and sum(sections) != rot_dim // 2):
            raise Qw35Error(f"rot_dim={rot_dim} must be a positive multiple of 16 and twice the sections {sections}")
        host = torch.empty(rot_dim // 2, dtype=torch.int64)
        _ffi.call("qw35_hip_rope_freq", rot_dim, float(base), C.c_void_p(host.data_ptr()))
        self.freq = host.to(device)  # 64-bit fixed-point turns per position
        self.rot_dim, self.sections, self.interleaved = rot_dim, sections, bool(interleaved)
        self.axes = max([i + 1 for i, s in enumerate(sections) if s], default=1)
        self.view = _ffi.Rope(self.freq.data_ptr(), rot_dim, int(interleaved),
                              (C.c_uint32 * 4)(*(sections + [0] * (4 - len(sections)))))
        self._at = C.addressof(self.view)


def _turn(rope: Rotary | None, positions, n: int, device: int) -> tuple:
    """The rope, positions and n_axes arguments of a call."""
    if rope is None:
        return None, None, 0
    if positions is None:
        raise Qw35Error("positions are needed with a rope")
    if rope.freq.get_device() != device:
        raise Qw35Error(f"the rope lives on {rope.freq.device}, the input on cuda:{device}")
    if positions.dim() == 1:
        return rope._at, _index(positions, torch.int32, (n,), device, "positions"), 1
    axes = int(positions.shape[0])
    if axes != 1 and axes != rope.axes:
        raise Qw35Error(f"positions have {axes} axes, the sections 1 or {rope.axes}")
    return rope._at, _index(positions, torch.int32, (axes, n), device, "positions"), axes


def rotate(x: torch.Tensor, rope: Rotary | None, positions: torch.Tensor | None = None, norm: torch.Tensor | None = None,
           eps: float = 1e-6, out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
           stream=None) -> torch.Tensor:
    """RMS norm (with ``norm``, fp32 [dim]) and rotation of x [n_tokens, heads, dim].

    x: fp32, bf16 or fp16, any token and head stride; ``positions`` int32
    [n_tokens], or [axes, n_tokens] for the rope's sections.  Statistics and
    rotation in fp32, rounded once to ``out_dtype`` (default: ``out``'s or x's
    type).  ``out`` may be x."""
    if stream is not None:
        with _behind(stream, x):
            return rotate(x, rope, positions, norm, eps, out, out_dtype)
    device = x.get_device()
    if _elsewhere(device):
        with torch.cuda.device(device):
            return rotate(x, rope, positions, norm, eps, out, out_dtype)
    hx = _heads(x, "x")
    n, heads, dim = x.shape
    out = _output(out, out_dtype, x)
    hy = _heads(out, "out")
    weight = _vector(norm, dim, device, "norm")
    turn, pos, axes = _turn(rope, positions, n, device)
    if n:
        _call("qw35_hip_rotate", _HEADS.pack(*hx), _HEADS.pack(*hy), n, heads, dim, turn, pos, axes, weight, eps,
              rt._raw_stream(device))
    return out


class PagedCache:
    """A paged key/value cache of one layer (``qw35_hip_kv_cache``) over two tensors:

    k [n_pages, kv_heads, page_size / 32, dim / 8, 32, 8] and
    v [n_pages, kv_heads, page_size / 8, dim, 8], fp16, bf16 or float8_e4m3fn
    (then with an fp32 scale per kv head, default 1).  Slot ``s`` is token
    ``s % page_size`` of page ``s // page_size``.

    With scales fp32 [n_pages, kv_heads, page_size / 32] the cache is block-scaled,
    float8_e4m3fn or int8: the 32 tokens of a head with one ``s // 32`` have a scale
    of their own, for keys and for values, which ``kv_append`` writes (0 for a block
    of zeros, as a new cache's)."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None):
        if k.dim() != 6 or tuple(k.shape[4:]) != (32, 8) or not k.is_cuda or not k.is_contiguous():
            raise Qw35Error("cache keys must be a contiguous [n_pages, kv_heads, page_size / 32, dim / 8, 32, 8] device "
                            f"tensor, got {list(k.shape)}")
        pages, heads, blocks, octets = (int(s) for s in k.shape[:4])
        want = (pages, heads, blocks * 4, octets * 8, 8)
        if tuple(v.shape) != want or v.dtype != k.dtype or v.device != k.device or not v.is_contiguous():
            raise Qw35Error(f"cache values must be a contiguous {k.dtype} {list(want)} tensor on {k.device}")
        self.block_scales = k.dtype == torch.int8 or any(s is not None and s.dim() == 3 for s in (k_scale, v_scale))
        codes = _BLOCKS if self.block_scales else _CACHE
        if k.dtype not in codes:
            raise Qw35Error(f"a cache is float16, bfloat16 or float8_e4m3fn, with block scales float8_e4m3fn or int8, "
                            f"got {k.dtype}")
        if k.dtype != torch.float8_e4m3fn and not self.block_scales and (k_scale is not None or v_scale is not None):
            raise Qw35Error("only a float8_e4m3fn cache has scales")
        device = k.get_device()
        if self.block_scales:
            if k_scale is None or v_scale is None:
                raise Qw35Error(f"a block-scaled cache needs k_scale and v_scale [{pages}, {heads}, {blocks}]")
            at_k = _index(k_scale, torch.float32, (pages, heads, blocks), device, "k_scale")
            at_v = _index(v_scale, torch.float32, (pages, heads, blocks), device, "v_scale")
        else:
            at_k, at_v = _vector(k_scale, heads, device, "k_scale"), _vector(v_scale, heads, device, "v_scale")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.n_pages, self.kv_heads, self.page_size, self.head_dim = pages, heads, blocks * 32, octets * 8
        self.view = _ffi.KvCache(k.data_ptr(), v.data_ptr(), at_k, at_v, pages, self.page_size, heads, self.head_dim,
                                 codes[k.dtype], 0)
        self._at, self._device = C.addressof(self.view), device
        self.number = torch.float16 if k.dtype.itemsize == 1 else k.dtype  # that its elements are read as

    @classmethod
    def empty(cls, n_pages: int, kv_heads: int, page_size: int, head_dim: int, dtype: torch.dtype = torch.float16,
              k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None, device="cuda",
              block_scales: bool = False) -> "PagedCache":
        """A new cache; block-scaled (int8, or float8_e4m3fn with ``block_scales``) of zeros."""
        if page_size <= 0 or page_size % 32 or head_dim not in (64, 128, 256):
            raise Qw35Error(f"page_size={page_size} must be a multiple of 32 and head_dim={head_dim} 64, 128 or 256")
        shapes = ((n_pages, kv_heads, page_size // 32, head_dim // 8, 32, 8), (n_pages, kv_heads, page_size // 8, head_dim, 8))
        if block_scales or dtype == torch.int8:
            if k_scale is not None or v_scale is not None:
                raise Qw35Error("a new block-scaled cache makes its own scales")
            if dtype not in _BLOCKS:
                raise Qw35Error(f"a cache is float8_e4m3fn or int8 with block scales, got {dtype}")
            k, v = (torch.zeros(s, dtype=torch.uint8, device=device).view(dtype) for s in shapes)
            k_scale, v_scale = (torch.zeros((n_pages, kv_heads, page_size // 32), device=device) for _ in range(2))
        else:
            k, v = (torch.empty(s, dtype=dtype, device=device) for s in shapes)
        return cls(k, v, k_scale, v_scale)

    def slots(self, pages: torch.Tensor, at: torch.Tensor) -> torch.Tensor:
        """Slots of the tokens ``at`` (int tensor) of a sequence with page list ``pages``."""
        at = at.long()
        return pages.long()[at // self.page_size] * self.page_size + at % self.page_size


def kv_append(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, rope: Rotary | None = None,
              positions: torch.Tensor | None = None, norm: torch.Tensor | None = None, eps: float = 1e-6,
              stream=None) -> None:
    """Keys (normed and rotated as ``rotate`` does) and values [n_tokens, kv_heads,
    head_dim] into ``slots`` (int64 [n_tokens]; a negative one leaves its token out).

    Into an e4m3 cache go the values over the head's scale, rounded to nearest
    even, past +-448 to +-448.  In a block-scaled cache a block's scale doubles until
    the tokens fit its largest code (448, 127), and what the block held is rounded to
    it; writing a block's first token begins the block anew, at the least power of
    two, with its other tokens zero (``qw35_hip_kv_append`` has the details)."""
    if stream is not None:
        with _behind(stream, k):
            return kv_append(cache, k, v, slots, rope, positions, norm, eps)
    device = cache._device
    if _elsewhere(device):
        with torch.cuda.device(device):
            return kv_append(cache, k, v, slots, rope, positions, norm, eps)
    hk, hv = _heads(k, "k"), _heads(v, "v")
    n = int(k.shape[0])
    if k.shape != (n, cache.kv_heads, cache.head_dim) or v.shape != k.shape or k.dtype != v.dtype:
        raise Qw35Error(f"k and v must be [n_tokens, {cache.kv_heads}, {cache.head_dim}] of one type, got "
                        f"{list(k.shape)} {k.dtype} and {list(v.shape)} {v.dtype}")
    if k.get_device() != device or v.get_device() != device:
        raise Qw35Error(f"k and v must be on the cache's {cache.k.device}")
    where = _index(slots, torch.int64, (n,), device, "slots")
    weight = _vector(norm, cache.head_dim, device, "norm")
    turn, pos, axes = _turn(rope, positions, n, device)
    if n:
        _call("qw35_hip_kv_append", cache._at, _HEADS.pack(*hk), _HEADS.pack(*hv), n, where, turn, pos, axes, weight,
              eps, rt._raw_stream(device))


def kv_read(cache: PagedCache, slots: torch.Tensor, dtype: torch.dtype | None = None, k: torch.Tensor | None = None,
            v: torch.Tensor | None = None, stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values [n_tokens, kv_heads, head_dim] in ``slots`` (int64
    [n_tokens], repeats allowed; zeros for a negative one or one past the cache): the
    cache's elements times their scales, rounded once to ``dtype`` (fp32, bf16 or
    fp16; default ``k``'s type, else the cache's, fp16 of an 8-bit one).  Into ``k``
    and ``v`` where they are given, any token and head stride."""
    if stream is not None:
        with _behind(stream, slots):
            return kv_read(cache, slots, dtype, k, v)
    device = cache._device
    if _elsewhere(device):
        with torch.cuda.device(device):
            return kv_read(cache, slots, dtype, k, v)
    if slots.dim() != 1:
        raise Qw35Error("slots must be int64 [n_tokens]")
    n = slots.shape[0]
    where = _index(slots, torch.int64, (n,), device, "slots")
    heads, dim = cache.kv_heads, cache.head_dim
    shape = (n, heads, dim)
    if k is None and v is None:  # (rows of its own: what there is to check is the type)
        dtype = dtype or cache.number
        code = _FLOAT.get(dtype)
        if code is None:
            raise Qw35Error(f"dtype must be fp32, bf16 or fp16, got {dtype}")
        k = torch.empty(shape, dtype=dtype, device=cache.k.device)
        v = torch.empty_like(k)
        hk, hv = ((x.data_ptr(), heads * dim, dim, code, 0) for x in (k, v))
    else:
        dtype = dtype or (v if k is None else k).dtype
        k, v = (torch.empty(shape, dtype=dtype, device=cache.k.device) if x is None else x for x in (k, v))
        for name, x in (("k", k), ("v", v)):
            if x.shape != shape or x.dtype != dtype or x.get_device() != device:
                raise Qw35Error(f"{name} must be a {dtype} {list(shape)} tensor on {cache.k.device}, got {x.dtype} "
                                f"{list(x.shape)} on {x.device}")
        hk, hv = _heads(k, "k"), _heads(v, "v")
    if n:
        _call("qw35_hip_kv_read", cache._at, _HEADS.pack(*hk), _HEADS.pack(*hv), n, where, rt._raw_stream(device))
    return k, v


def _workspace_bytes(cache: PagedCache, n_heads: int, n_seqs: int, n_tokens: int) -> int:
    size = int(_ffi.load().qw35_hip_prefix_attention_workspace_size(C.byref(cache.view), n_heads, n_seqs, n_tokens))
    if size == 0:
        raise Qw35Error(f"prefix_attention: no workspace for n_heads={n_heads}, n_seqs={n_seqs}, n_tokens={n_tokens}")
    return size


def prefix_attention_workspace(cache: PagedCache, n_heads: int, n_seqs: int, n_tokens: int, device="cuda") -> torch.Tensor:
    """A workspace for ``prefix_attention`` of up to this batch (its contents do not
    matter; calls that overlap need one each)."""
    return torch.empty(_workspace_bytes(cache, n_heads, n_seqs, n_tokens), dtype=torch.uint8, device=device)


def prefix_attention(q: torch.Tensor, cache: PagedCache, pages: torch.Tensor, lengths: torch.Tensor,
                     starts: torch.Tensor | None = None, max_new: int = 0, prefix_pages: torch.Tensor | None = None,
                     prefix_len: int = 0, scale: float | None = None, window: int = 0, sink: int = 0,
                     gate: torch.Tensor | None = None, out: torch.Tensor | None = None,
                     out_dtype: torch.dtype | None = None, workspace: torch.Tensor | None = None,
                     stream=None) -> torch.Tensor:
    """Attention of the new tokens q [n_tokens, n_heads, head_dim] of a batch of sequences.

    Sequence s has the new tokens ``starts[s]:starts[s + 1]`` (int32 [n_seqs + 1];
    None: one each), the last of its ``lengths[s]`` own tokens (int32), which lie in
    the pages ``pages[s]`` (int32 [n_seqs, pages_per_seq]) after the ``prefix_len``
    tokens in ``prefix_pages`` that all sequences share.  A token sees the
    positions up to its own, with ``window`` only the last ``window`` of them and
    the first ``sink``.  Result: softmax(scale q k) v (scale default
    1 / sqrt(head_dim)), zeros where nothing is seen, times sigmoid(``gate``), in
    ``out_dtype`` (default q's type); the softmax' weights have q's precision in the
    product with v whatever ``out_dtype`` is, everything else is fp32.

    q has the cache's type; over an e4m3 cache either 16-bit type, over an int8 one
    fp16.

    ``max_new``: the most new tokens of a sequence, where it is known: it chooses
    how rows are divided, not what is computed.  All lengths live on the device, so
    a recorded call serves every later step."""
    if stream is not None:
        with _behind(stream, q):
            return prefix_attention(q, cache, pages, lengths, starts, max_new, prefix_pages, prefix_len, scale, window,
                                    sink, gate, out, out_dtype, workspace)
    device = cache._device
    if _elsewhere(device):
        with torch.cuda.device(device):
            return prefix_attention(q, cache, pages, lengths, starts, max_new, prefix_pages, prefix_len, scale, window,
                                    sink, gate, out, out_dtype, workspace)
    hq = _heads(q, "q")
    n, heads, dim = q.shape
    if dim != cache.head_dim or q.get_device() != device:
        raise Qw35Error(f"q must be [n_tokens, n_heads, {cache.head_dim}] on {cache.k.device}, got {list(q.shape)}")
    if lengths.dim() != 1 or pages.dim() != 2:
        raise Qw35Error("lengths must be int32 [n_seqs], pages int32 [n_seqs, pages_per_seq]")
    seqs, per_seq = pages.shape
    at_lengths = _index(lengths, torch.int32, (seqs,), device, "lengths")
    at_pages = _index(pages, torch.int32, (seqs, per_seq), device, "pages")
    at_starts = 0 if starts is None else _index(starts, torch.int32, (seqs + 1,), device, "starts")
    if prefix_len and prefix_pages is None:
        raise Qw35Error("prefix_len needs prefix_pages")
    at_prefix = shared = 0
    if prefix_pages is not None:
        shared = prefix_pages.numel()
        at_prefix = _index(prefix_pages, torch.int32, (shared,), device, "prefix_pages")
    if max_new < 0 or prefix_len < 0 or window < 0 or sink < 0:
        raise Qw35Error("max_new, prefix_len, window and sink cannot be negative")
    out = _output(out, out_dtype, q)
    ho = _heads(out, "out")
    hg = _NO_HEADS
    if gate is not None:
        if gate.shape != q.shape or gate.get_device() != device:
            raise Qw35Error(f"gate must be a {list(q.shape)} tensor on {q.device}")
        hg = _heads(gate, "gate")
    if n == 0:
        return out
    if workspace is None:  # this call's own
        workspace = prefix_attention_workspace(cache, heads, seqs, n, device=q.device)
    if workspace.get_device() != device or not workspace.is_contiguous():
        raise Qw35Error(f"workspace must be a contiguous tensor on {q.device}")
    if not prefix_len:
        at_prefix = shared = 0
    try:
        op = _ATTENTION.pack(*hq, *ho, *hg, n, heads, seqs, max_new, at_starts, at_lengths, at_pages, at_prefix, per_seq,
                             shared, prefix_len, window, sink, 1.0 / math.sqrt(dim) if scale is None else scale,
                             workspace.data_ptr(), workspace.nbytes)
    except (struct.error, OverflowError) as e:
        raise Qw35Error(f"prefix_attention: max_new, prefix_len, window, sink or scale out of range: {e}") from None
    _call("qw35_hip_prefix_attention", op, cache._at, rt._raw_stream(device))
    return out


class GatedAttention:
    """One attention layer between its input norm and the residual stream, as the
    reference records it (Qw35MetalRuntime+Attention.m:13-117): the q / k / v
    projections, ``rotate`` of the queries, ``kv_append``, ``prefix_attention``
    with the output gate and the output projection added to the residual.

    ``weights``: ``attn_q`` (heads x [queries, then gates] if the rows are twice
    heads x dim, else queries only), ``attn_k``, ``attn_v`` and ``attn_output`` as
    ``HipWeight``.  Up to 8 tokens run the decode GEMVs, more the prefill matmul
    (fp32 activations).  Nothing of a call is kept but the cache, workspaces
    included (torch's allocator serves them): calls of one layer may overlap on
    several streams as far as their slots differ (their blocks of 32, of a
    block-scaled cache), and a call can be recorded into a graph, with lengths, slots,
    positions and pages on the device."""

    def __init__(self, weights: dict, cache: PagedCache, heads: int, rope: Rotary | None,
                 q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, eps: float = 1e-6,
                 max_seqs: int = 8, max_tokens: int = 8, window: int = 0, sink: int = 0):
        dim, q_rows = cache.head_dim, weights["attn_q"].rows
        self.gated = q_rows == 2 * heads * dim
        kv = cache.kv_heads * dim
        if q_rows not in (heads * dim, 2 * heads * dim) or weights["attn_k"].rows != kv or weights["attn_v"].rows != kv:
            raise Qw35Error(f"attn_q, attn_k and attn_v have {q_rows}, {weights['attn_k'].rows} and "
                            f"{weights['attn_v'].rows} rows for {heads} heads and {cache.kv_heads} kv heads of {dim}")
        if weights["attn_output"].k != heads * dim:
            raise Qw35Error(f"attn_output has {weights['attn_output'].k} columns for {heads} heads of {dim}")
        self.weights, self.cache, self.heads, self.rope, self.eps = weights, cache, heads, rope, eps
        self.q_norm, self.k_norm, self.window, self.sink = q_norm, k_norm, window, sink
        # an e4m3 cache takes either 16-bit type: fp16 keeps more of a normed query
        self.q_dtype = torch.float16 if cache.k.dtype.itemsize == 1 else cache.k.dtype
        self.max_seqs, self.max_tokens = max_seqs, max_tokens
        self.workspace_bytes = _workspace_bytes(cache, heads, max_seqs, max_tokens)
        if max_tokens > _ffi.MAX_BATCH:
            for w in weights.values():
                w.prefill  # (a k-quant's fp16 image, here and not in a call)

    def _project(self, name: str, x: torch.Tensor) -> torch.Tensor:
        w = self.weights[name]
        if x.shape[0] <= _ffi.MAX_BATCH:
            return rt.decode_matvec(w, x)
        return rt.matmul_prefill(w.prefill, x, out_dtype=torch.float32)

    def __call__(self, x: torch.Tensor, residual: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
                 pages: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor | None = None, max_new: int = 0,
                 prefix_pages: torch.Tensor | None = None, prefix_len: int = 0, stream=None) -> torch.Tensor:
        """Adds the layer's output for the normed inputs x (fp32 [n_tokens, embedding])
        to ``residual`` (fp32, same shape) and returns it.  ``slots`` are the new
        tokens' places in the cache, the other arguments ``rotate``'s and
        ``prefix_attention``'s (``lengths`` count the new tokens)."""
        if stream is not None:
            with _behind(stream, x):
                return self(x, residual, positions, slots, pages, lengths, starts, max_new, prefix_pages, prefix_len)
        if _elsewhere(self.cache._device):
            with torch.cuda.device(self.cache._device):
                return self(x, residual, positions, slots, pages, lengths, starts, max_new, prefix_pages, prefix_len)
        n, dim, cache = int(x.shape[0]), self.cache.head_dim, self.cache
        if n > self.max_tokens or lengths.shape[0] > self.max_seqs:
            raise Qw35Error(f"{n} tokens of {lengths.shape[0]} sequences are over the layer's {self.max_tokens} and "
                            f"{self.max_seqs}")
        if x.get_device() != cache._device:
            raise Qw35Error(f"x must be on the cache's {cache.k.device}, got {x.device}")
        if (residual.shape != x.shape or residual.dtype != torch.float32 or not residual.is_contiguous()
                or residual.device != x.device):
            raise Qw35Error(f"residual must be a contiguous fp32 {list(x.shape)} tensor on {x.device}")
        if n == 0:
            return residual
        q = self._project("attn_q", x).view(n, self.heads, -1)
        k = self._project("attn_k", x).view(n, cache.kv_heads, dim)
        v = self._project("attn_v", x).view(n, cache.kv_heads, dim)
        turned = rotate(q[..., :dim], self.rope, positions, norm=self.q_norm, eps=self.eps, out_dtype=self.q_dtype)
        kv_append(cache, k, v, slots, rope=self.rope, positions=positions, norm=self.k_norm, eps=self.eps)
        core = prefix_attention(turned, cache, pages, lengths, starts, max_new=max_new, prefix_pages=prefix_pages,
                                prefix_len=prefix_len, window=self.window, sink=self.sink,
                                gate=q[..., dim:] if self.gated else None, out_dtype=torch.float32,
                                workspace=torch.empty(self.workspace_bytes, dtype=torch.uint8, device=x.device)).view(n, -1)
        out = self.weights["attn_output"]
        if n <= _ffi.MAX_BATCH:
            rt.decode_matvec(out, core, dst=residual, residual=True)
        else:
            rt.matmul_prefill(out.prefill, core, out_dtype=torch.float32, dst=residual, epilogue=_ffi.EPILOGUE_ADD)
        return residual

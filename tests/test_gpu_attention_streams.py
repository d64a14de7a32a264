"""The attention operators and the layer on another stream than the current one:
behind what the current stream holds, with temporaries that no other stream is
given before the call is done."""
from __future__ import annotations

import pytest
import torch

from tests import attention_reference as ref
from tests.test_gpu_attention import E4M3, F16, Batch, _cache, _gen
from tests.test_gpu_gated_attention import DIM, E, KV, _layer
from tests.test_gpu_streams import _busy, _made_on

pytestmark = pytest.mark.gpu


def _fill_free_memory(*sizes):
    """Takes and fills whatever blocks of those sizes the current stream's memory has."""
    for size in sizes:
        for t in [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(8)]:
            t.fill_(0xff)


def test_operators_run_behind_the_current_stream(cuda):
    """Inputs that the current stream still makes are there."""
    from qwowl35_amd import attention as at

    randn = _gen(cuda, 1)
    x, k, v = randn(5, 4, 64), randn(5, 2, 64), randn(5, 2, 64)
    pos, slots = torch.arange(5, dtype=torch.int32, device=cuda), torch.arange(5, device=cuda)
    rope = at.Rotary(64, 1e4, device=cuda)
    pages, lengths = torch.zeros(1, 1, dtype=torch.int32, device=cuda), torch.tensor([5], dtype=torch.int32, device=cuda)
    starts = torch.tensor([0, 5], dtype=torch.int32, device=cuda)
    here, there = (_cache(cuda, 1, 2, 32, 64, F16) for _ in range(2))

    def step(cache, x, k, stream):
        q = at.rotate(x, rope, pos, out_dtype=F16, stream=stream)
        at.kv_append(cache, k, v, slots, rope, pos, stream=stream)
        return q, at.prefix_attention(q, cache, pages, lengths, starts, stream=stream)

    want = step(here, x, k, None)
    late_x, late_k, side = torch.full_like(x, 3.0), torch.full_like(k, 3.0), torch.cuda.Stream()
    torch.cuda.synchronize()
    _busy()
    late_x.copy_(x)
    late_k.copy_(k)
    got = step(there, late_x, late_k, side)
    torch.cuda.synchronize()
    assert torch.equal(here.k[:, :, 0, :, :5], there.k[:, :, 0, :, :5])
    for a, b in zip(got, want):
        assert torch.equal(a, b) and _made_on(a) == side.cuda_stream


@pytest.mark.parametrize("cache", [F16, E4M3])
def test_attention_keeps_its_own_workspace(cuda, cache):
    """A call without a workspace, waiting on its stream, while the current stream takes and fills memory."""
    from qwowl35_amd import attention as at

    b = Batch(cuda, [1, 3, 1], [500, 3, 77], 900, 8, 2, 64, 64, F16, cache, seed=2)
    want, bound = b.want()
    size = at.prefix_attention_workspace(b.cache, 8, 3, 5).numel()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        _busy()
    got = b.run(stream=side, workspace=None)
    _fill_free_memory(size, size)
    torch.cuda.synchronize()
    ref.close(got, want, bound, "a workspace of the call")


@pytest.mark.parametrize("tokens", [2, 20])  # decode GEMVs, prefill matmuls
def test_layer_on_another_stream(cuda, tokens):
    """The layer waiting on its stream: its projections, queries and result stay its own, and are not cleared late."""
    layer, rand = _layer(cuda, True, F16)
    other, _ = _layer(cuda, True, F16)
    x, n = rand(tokens, E), torch.arange(tokens, device=cuda, dtype=torch.int32)
    pages, lengths = torch.tensor([[1]], dtype=torch.int32, device=cuda), torch.tensor([tokens], dtype=torch.int32, device=cuda)
    starts = torch.tensor([0, tokens], dtype=torch.int32, device=cuda)
    slots = layer.cache.slots(pages[0], n)
    want = layer(x, torch.zeros_like(x), n, slots, pages, lengths, starts)
    late, res, side = torch.zeros_like(x), torch.full_like(x, 9.0), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        _busy()
    _busy()
    late.copy_(x)
    res.zero_()
    got = other(late, res, n, slots, pages, lengths, starts, stream=side)
    rows = tokens * DIM * 4
    _fill_free_memory(rows * 8, rows * KV, rows * 4, rows * 2)
    torch.cuda.synchronize()
    assert got is res and torch.equal(got, want)


def test_the_current_stream_by_argument(cuda):
    b = Batch(cuda, [1, 2], [33, 64], 20, 4, 2, 64, 32, F16, F16, seed=12)
    want = b.run()
    assert torch.equal(b.run(stream=torch.cuda.current_stream()), want)


@pytest.mark.parametrize("tokens", [3, 20])
def test_overlapping_calls_of_one_layer(cuda, tokens, monkeypatch):
    """Calls of a layer on several streams at a time, over pages of their own: no two have a workspace in common."""
    from qwowl35_amd import attention as at
    from qwowl35_amd import runtime as rt

    layer, rand = _layer(cuda, True, F16)
    other, _ = _layer(cuda, True, F16)
    n = torch.arange(tokens, device=cuda, dtype=torch.int32)
    lengths, starts = (torch.tensor(v, dtype=torch.int32, device=cuda) for v in ([tokens], [0, tokens]))
    pages = [torch.tensor([[p]], dtype=torch.int32, device=cuda) for p in (1, 4, 6)]
    slots = [layer.cache.slots(p[0], n) for p in pages]
    x, res = [rand(tokens, E) for _ in pages], [torch.zeros(tokens, E, device=cuda) for _ in pages]
    want = [other(x[i], torch.zeros_like(x[i]), n, slots[i], p, lengths, starts) for i, p in enumerate(pages)]
    used, attend, make = [], at.prefix_attention, rt.prefill_workspace
    monkeypatch.setattr(at, "prefix_attention", lambda *a, **k: (used.append(k["workspace"]), attend(*a, **k))[1])
    monkeypatch.setattr(rt, "prefill_workspace", lambda *a, **k: (used.append(make(*a, **k)), used[-1])[1])
    streams = [torch.cuda.Stream() for _ in pages]
    torch.cuda.synchronize()
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            _busy()
            layer(x[i], res[i], n, slots[i], pages[i], lengths, starts)
    torch.cuda.synchronize()
    for got, w in zip(res, want):
        assert torch.equal(got, w)
    assert len({t.data_ptr() for t in used}) == len(used) == (3 if tokens <= 8 else 15)


def test_a_chunk_has_the_workspace_of_its_own_size(cuda, monkeypatch):
    """A chunk of 90 tokens splits an 8192 x 4096 product further than one of 96: it has the room that it asks for."""
    import ctypes as C

    from qwowl35_amd import _ffi
    from qwowl35_amd import attention as at
    from qwowl35_amd import runtime as rt

    heads, kv, dim, wide = 16, 4, 256, 4096
    g = torch.Generator(device=cuda)
    g.manual_seed(4)
    weights = {n: rt.quantize_weight(torch.randn(rows, wide, generator=g, device=cuda) * 0.02, rt.TYPE_Q8_0)
               for n, rows in (("attn_q", 2 * heads * dim), ("attn_k", kv * dim), ("attn_v", kv * dim), ("attn_output", wide))}
    layer = at.GatedAttention(weights, at.PagedCache.empty(2, kv, 96, dim, device=cuda), heads, None, max_tokens=96)
    made, run = [], rt.matmul_prefill
    monkeypatch.setattr(rt, "matmul_prefill", lambda w, a, **k: (made.append((w, k.get("workspace", True))),
                                                                 run(w, a, **k))[1])
    n = torch.arange(90, device=cuda, dtype=torch.int32)
    pages, x = torch.tensor([[1]], dtype=torch.int32, device=cuda), torch.randn(90, wide, device=cuda)
    lengths, starts = (torch.tensor(v, dtype=torch.int32, device=cuda) for v in ([90], [0, 90]))
    layer(x, torch.zeros_like(x), n, layer.cache.slots(pages[0], n), pages, lengths, starts)
    assert len(made) == 4
    for w, ws in made:  # (True: of this call's size)
        need = int(_ffi.load().qw35_hip_matmul_prefill_workspace_size(C.byref(w.view), 90))
        assert ws is True or ws.numel() >= need

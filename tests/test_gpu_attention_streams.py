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

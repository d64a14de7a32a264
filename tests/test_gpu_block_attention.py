"""Attention over a block-scaled cache against its formula in float64, at the
sizes, masks and scales where it can go wrong."""
from __future__ import annotations

import math

import pytest
import torch

from tests import attention_reference as ref
from tests.block_reference import BlockBatch, _gen, close
from tests.test_gpu_attention import BF16, E4M3, F16, F32, SHAPES

pytestmark = pytest.mark.gpu

I8 = torch.int8
KINDS = [(F16, I8), (F16, E4M3), (BF16, E4M3)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype,kind", KINDS)
def test_shapes(cuda, shape, dim, dtype, kind):
    new, lens, prefix, heads, kv_heads, page = SHAPES[shape]
    b = BlockBatch(cuda, new, lens, prefix, heads, kv_heads, dim, page, dtype, kind, seed=len(shape) + dim)
    want, bound = b.want()
    got = b.run()
    assert got.dtype == dtype
    close(got, want, bound, shape)
    close(b.run(out_dtype=F32, max_new=0), want, bound, shape + " in fp32, rows divided for any sequence")


@pytest.mark.parametrize("window,sink", [(1, 0), (33, 0), (40, 5), (64, 64), (500, 3), (7, 400)])
@pytest.mark.parametrize("shape", ["prefix", "chunk", "rows_60", "tile_edges", "late"])
@pytest.mark.parametrize("dim,dtype,kind", [(64, BF16, E4M3), (128, F16, E4M3), (256, F16, I8), (64, F16, I8)])
def test_window_and_sink(cuda, window, sink, shape, dim, dtype, kind):
    new, lens, prefix, heads, kv_heads, page = SHAPES[shape]
    b = BlockBatch(cuda, new, lens, prefix, heads, kv_heads, dim, page, dtype, kind, seed=window + dim)
    want, bound = b.want(window=window, sink=sink)
    close(b.run(window=window, sink=sink), want, bound, f"{shape} window {window} sink {sink}")


@pytest.mark.parametrize("gate", [F32, F16, BF16])
@pytest.mark.parametrize("shape", ["one", "prefix", "chunk"])
def test_gate(cuda, gate, shape):
    new, lens, prefix, heads, kv_heads, page = SHAPES[shape]
    b = BlockBatch(cuda, new, lens, prefix, heads, kv_heads, 128, page, F16, I8, seed=4)
    g = (_gen(cuda, 8)(b.q.shape[0], heads, 256) * 3).to(gate)[..., 128:]
    want, bound = b.want(gate=g)
    close(b.run(gate=g), want, bound, "gate")


@pytest.mark.parametrize("dim,dtype,kind", [(64, F16, I8), (128, F16, I8), (256, F16, I8), (256, BF16, E4M3)])
def test_many_pieces(cuda, dim, dtype, kind):
    """Over 64 tiles a wave (their scales are looked up anew), pieces over the whole grid."""
    b = BlockBatch(cuda, [1, 3, 1], [5000, 1, 777], 9000, 8, 2, dim, 64, dtype, kind, seed=2)
    want, bound = b.want()
    close(b.run(), want, bound, "many pieces")
    c = BlockBatch(cuda, [1], [70001], 0, 1, 1, dim, 4096, dtype, kind, seed=3)
    want, bound = c.want()
    close(c.run(), want, bound, "one long sequence")


@pytest.mark.parametrize("dim,dtype,kind", [(64, F16, I8), (128, BF16, E4M3), (256, F16, I8), (256, F16, E4M3)])
def test_long_chunks(cuda, dim, dtype, kind):
    """Shared tiles over more than 64 of them, rows of which some see a part."""
    b = BlockBatch(cuda, [200], [2500], 3000, 4, 2, dim, 96, dtype, kind, seed=7)
    want, bound = b.want()
    close(b.run(), want, bound, "a chunk over a prefix")
    want, bound = b.want(window=700, sink=33)
    close(b.run(window=700, sink=33), want, bound, "under a window")


@pytest.mark.parametrize("dim,dtype,kind", [(64, F16, I8), (64, BF16, E4M3), (256, F16, I8)])
def test_many_sequences(cuda, dim, dtype, kind):
    """More sequences than a line of lanes, and than are kept in LDS, with a prefix and without."""
    for seqs, prefix in ((70, 40), (300, 33), (300, 0)):
        b = BlockBatch(cuda, [1 + (s % 90 == 0) for s in range(seqs)], [2 + 7 * s % 95 for s in range(seqs)], prefix, 2, 1,
                       dim, 32, dtype, kind, seed=seqs + prefix)
        want, bound = b.want()
        close(b.run(), want, bound, f"{seqs} sequences after {prefix}")


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("shape", ["prefix", "chunk", "chunk_long"])
def test_scales_far_apart(cuda, dtype, kind, shape):
    """Values of one block 2^100 times another's: a row has what it sees, whatever lies beside it."""
    new, lens, prefix, heads, kv_heads, page = SHAPES[shape]
    b = BlockBatch(cuda, new, lens, prefix, heads, kv_heads, 128, page, dtype, kind, seed=5)
    g = torch.Generator(device=cuda).manual_seed(1)
    e = torch.randint(-50, 50, b.cache.v_scale.shape, generator=g, device=cuda)
    b.cache.v_scale.mul_(torch.exp2(e.float()))
    b.cache.k_scale.mul_(torch.exp2(torch.randint(-20, 1, e.shape, generator=g, device=cuda).float()))
    want, bound = b.want()
    close(b.run(out_dtype=F32), want, bound, "scales far apart")


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("shape", ["one", "prefix", "chunk", "rows_60"])
def test_scales_that_are_no_powers_of_two(cuda, dtype, kind, shape):
    new, lens, prefix, heads, kv_heads, page = SHAPES[shape]
    b = BlockBatch(cuda, new, lens, prefix, heads, kv_heads, 64, page, dtype, kind, seed=6)
    for s in (b.cache.k_scale, b.cache.v_scale):
        s.mul_(torch.rand(s.shape, device=cuda) + 0.6)
    want, bound = b.want()
    close(b.run(), want, bound, "any scales")


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("shape", ["one", "tile_edges", "prefix", "chunk", "chunk_long"])
@pytest.mark.parametrize("share", [0.5, 1.0])
def test_blocks_of_zeros(cuda, dtype, kind, shape, share):
    """A scale of zero makes a block's tokens zero: they count in the softmax, and their values are zero."""
    new, lens, prefix, heads, kv_heads, page = SHAPES[shape]
    b = BlockBatch(cuda, new, lens, prefix, heads, kv_heads, 128, page, dtype, kind, seed=9)
    g = torch.Generator(device=cuda).manual_seed(3)
    for s in (b.cache.k_scale, b.cache.v_scale):
        s.masked_fill_(torch.rand(s.shape, generator=g, device=cuda) < share, 0.0)
    if kind == E4M3:  # (NaN times zero is NaN: unseen slots are kept out by their place)
        assert b.cache.k.view(torch.uint8).eq(0x7f).any()
    want, bound = b.want()
    close(b.run(out_dtype=F32), want, bound, "blocks of zeros")


def test_a_written_and_attended_cache(cuda):
    """Tokens appended one by one and in chunks, attended over after every call, as a decode loop does."""
    from qwowl35_amd import attention as at

    heads, kv, dim, page = 8, 2, 128, 64
    for kind in (I8, E4M3):
        c = at.PagedCache.empty(6, kv, page, dim, kind, device=cuda, block_scales=True)
        randn, pages = _gen(cuda, 12), torch.tensor([[4, 1, 5]], dtype=torch.int32, device=cuda)
        done = 0
        for new in (37, 1, 1, 30, 1, 50):
            t = torch.arange(done, done + new, device=cuda)
            k, v = randn(new, kv, dim) * (1 + done / 20), randn(new, kv, dim) * (1 + done / 9)
            at.kv_append(c, k, v, c.slots(pages[0], t))
            done += new
            q = randn(new, heads, dim).to(F16)
            got = at.prefix_attention(q, c, pages, torch.tensor([done], dtype=torch.int32, device=cuda),
                                      torch.tensor([0, new], dtype=torch.int32, device=cuda))
            kk, vv = at.kv_read(c, c.slots(pages[0], torch.arange(done, device=cuda)), dtype=F32)
            seen = torch.arange(done) <= done - new + torch.arange(new)[:, None]
            want, bound = ref.attend(q, kk, vv, seen, dim ** -0.5, F16)
            ref.close(got, want, bound * (1 + 2.0 ** -5), f"{kind} after {done} tokens")


def test_nan_of_an_e4m3_block_stays_where_it_is_seen(cuda):
    """A NaN value reaches the rows that see it, in its column, and no other."""
    b = BlockBatch(cuda, [20], [50], 0, 2, 1, 64, 64, F16, E4M3, seed=13)
    want, bound = b.want()
    slot = b.cache.slots(b.pages[0], torch.tensor([40], device=cuda))[0]
    page, at = int(slot) // 64, int(slot) % 64
    b.cache.v.view(torch.uint8)[page, 0, at // 8, 5, at % 8] = 0x7f
    got = b.run()
    bad = got.isnan()
    assert bad[10:, :, 5].all() and int(bad.sum()) == 10 * 2  # (the tokens 40..49 are the rows 10..19)
    keep = ~bad.cpu()
    keep[..., 5] = False
    ref.close(got.cpu()[keep], want[keep], bound[keep], "the other columns")


def test_negative_and_zero_softmax_scale(cuda):
    for scale in (-0.1, 0.0, 1e-30):
        b = BlockBatch(cuda, [3, 1], [70, 33], 40, 4, 2, 64, 32, F16, I8, seed=14)
        if scale == 0.0:  # every token alike
            b.q.zero_()
            want, bound = b.want()
            close(b.run(scale=0.0), want, bound, "scale 0")
            continue
        want, bound = b.want(scale=scale)
        close(b.run(scale=scale), want, bound, f"scale {scale}")


def test_queries_of_another_type_are_refused(cuda):
    from qwowl35_amd import Qw35Error

    b = BlockBatch(cuda, [1], [5], 0, 2, 1, 64, 32, F16, I8)
    b.q = b.q.to(BF16)
    with pytest.raises(Qw35Error, match="f16 for an i8 one"):
        b.run()
    assert math.isfinite(float(b.lengths.sum()))


def test_recorded_steps(cuda):
    """Append and attention of two sequences in one graph, replayed with eager work between, against eager steps."""
    from qwowl35_amd import attention as at

    kv, heads, dim, page = 2, 4, 128, 32
    mine, other = (at.PagedCache.empty(12, kv, page, dim, I8, device=cuda) for _ in range(2))
    randn = _gen(cuda, 15)
    pages = torch.tensor([[3, 1, 7], [8, 6, 0]], dtype=torch.int32, device=cuda)
    k, v, q = torch.zeros(2, kv, dim, device=cuda), torch.zeros(2, kv, dim, device=cuda), torch.zeros(2, heads, dim, dtype=F16, device=cuda)
    slots, lengths = torch.full((2,), -1, device=cuda), torch.ones(2, dtype=torch.int32, device=cuda)
    out = torch.empty_like(q)
    ws = at.prefix_attention_workspace(mine, heads, 2, 2)

    def step(c, to, ws=None):
        at.kv_append(c, k, v, slots)
        at.prefix_attention(q, c, pages, lengths, out=to, workspace=ws)
        return at.kv_read(c, slots)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(mine, out, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        read = step(mine, out, ws)
    for i in range(70):
        for x in (k, v):
            x.copy_(randn(2, kv, dim) * (1 + i / 10))
        q.copy_(randn(2, heads, dim))
        lengths.fill_(i + 1)
        slots.copy_(torch.stack([mine.slots(pages[s], torch.tensor(i, device=cuda)) for s in range(2)]))
        graph.replay()
        want = torch.empty_like(q)
        back = step(other, want)
        assert torch.equal(out, want) and torch.equal(read[0], back[0]) and torch.equal(read[1], back[1]), i
        if i % 10 == 0:
            torch.cuda.synchronize()
    for a, b in ((mine.k_scale, other.k_scale), (mine.v_scale, other.v_scale), (mine.k, other.k), (mine.v, other.v)):
        assert bool((a == b).all())

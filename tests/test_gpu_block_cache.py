"""The block-scaled cache: what an append makes of codes and scales, bit for bit
where the tokens come as they are, and reading back of every kind of cache."""
from __future__ import annotations

import math

import pytest
import torch

from tests import attention_reference as ref
from tests import block_reference as blk
from tests.test_gpu_attention import BF16, E4M3, F16, F32, _cache, _gen

pytestmark = pytest.mark.gpu

I8 = torch.int8


def _blocks(cuda, pages, heads, page, dim, kind, seed=1, **kw):
    from qwowl35_amd import attention as at

    c = at.PagedCache.empty(pages, heads, page, dim, kind, device=cuda, block_scales=True)
    torch.manual_seed(seed)
    blk.fill(c, _gen(cuda, seed), **kw)
    return c


CALLS = {  # the slots of each call, of pages of 64 or 96 tokens
    "one": lambda page: [[page + 5]],
    "decode": lambda page: [[i, page + 30 + i] for i in range(5)],              # two sequences, over a block's end
    "prompt": lambda page: [list(range(70)), [70], [71, 72]],
    "ragged": lambda page: [list(range(3, 30)), list(range(30, 37))],
    "order": lambda page: [[9, 40, 8, 10, 41, 11, 2 * page + 31, 39, 0, 2 * page, 64 % page, 17]],
    "padding": lambda page: [[-1, 0, 1, -1, 2, 10 ** 12, 3, 40, -5, 41, 3 * page, 4]],
    "twice": lambda page: [[5, 6, 5, 7, 5], [33, 33]],
    "rewrite": lambda page: [list(range(45)), [36], [32, 33], list(range(40, 50))],
}


@pytest.mark.parametrize("calls", CALLS)
@pytest.mark.parametrize("dim,heads,page", [(64, 3, 64), (128, 1, 96), (256, 4, 64)])
@pytest.mark.parametrize("dtype,kind", [(F32, I8), (BF16, I8), (F32, E4M3), (F16, E4M3)])
def test_append(cuda, calls, dim, heads, page, dtype, kind):
    """Calls that grow, begin anew and rewrite blocks; everything that no call names stays."""
    from qwowl35_amd import attention as at

    c = _blocks(cuda, 3, heads, page, dim, kind)
    want = blk.decode(c)
    randn = _gen(cuda, dim + len(calls))
    for i, slots in enumerate(CALLS[calls](page)):
        n = len(slots)
        k = (randn(n, heads, dim + 8) * 3.0 ** i).to(dtype)[..., :dim]
        v = (randn(heads, n, dim) * 5.0 ** i).to(dtype).transpose(0, 1)
        at.kv_append(c, k, v, torch.tensor(slots, device=cuda))
        for state, x in zip(want, (k, v)):
            blk.append(state, x.double().cpu(), slots, kind)
        blk.same(c, want, f"call {i}")


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("n,heads", [(300, 8), (2100, 1), (16384 + 40, 1)])
def test_append_of_many_tokens(cuda, kind, n, heads):
    """Workgroups that look for several blocks, and calls that are written in slices."""
    from qwowl35_amd import attention as at

    page, dim = 64, 64
    c = _blocks(cuda, n // page + 3, heads, page, dim, kind)
    want = blk.decode(c)
    randn = _gen(cuda, n)
    k, v = randn(n, heads, dim), randn(n, heads, dim)
    slots = torch.arange(n) + 21
    slots[100:140] = slots[100:140].flip(0)
    at.kv_append(c, k, v, slots.to(cuda))
    for first in range(0, n, 16384):
        for state, x in zip(want, (k, v)):
            blk.append(state, x[first:first + 16384].double().cpu(), slots[first:first + 16384], kind)
    blk.same(c, want)


MANY = {  # slots of n tokens, of pages of 64
    "step": lambda n: torch.arange(n) * 64 + 5,                                     # a decode step: a block for each
    "prompts": lambda n: torch.cat([p * 1024 + torch.arange(37 * p % 50, 37 * p % 50 + m)
                                    for p, m in enumerate((n // 3, n // 4 + 7, n - n // 3 - n // 4 - 7))]),
    "apart": lambda n: torch.arange(n) // 2 + torch.arange(n) % 2 * 2048,            # two sequences token by token
    "late": lambda n: torch.cat([torch.arange(n - 3), torch.tensor([7, 40, 7])]),    # a block's tokens at either end
    "shuffled": lambda n: torch.randperm(n, generator=torch.Generator().manual_seed(n)),
    "padded": lambda n: torch.where(torch.arange(n) % 40 < 33, torch.arange(n), -1),
    "one": lambda n: torch.arange(n) % 32 + 96,                                      # every token in one block
}


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("many", MANY)
@pytest.mark.parametrize("n", [64, 65, 130, 300, 700])
def test_append_wherever_the_tokens_go(cuda, kind, many, n):
    """Every block has one writer, which finds all of its tokens in the call."""
    from qwowl35_amd import attention as at

    slots = MANY[many](n)
    c = _blocks(cuda, int(slots.max()) // 64 + 2, 2, 64, 64, kind)
    want = blk.decode(c)
    randn = _gen(cuda, n)
    k, v = randn(n, 2, 64), randn(n, 2, 64)
    at.kv_append(c, k, v, slots.to(cuda))
    for state, x in zip(want, (k, v)):
        blk.append(state, x.double().cpu(), slots, kind)
    blk.same(c, want, many)


def _steps(n, step):
    """Slots of a step of n sequences, a page of 64 each, at different places; some without a token, some with two."""
    i = torch.arange(n)
    slots = i * 64 + (i * 7) % 31 + step
    slots[i % 23 == 5] = -1
    slots[n - 1] = slots[3] + (-1 if slots[3] % 32 else 1)   # block 3's other token, behind all
    slots[n // 2] = slots[10]                                # the last of two counts
    return slots


@pytest.mark.parametrize("n,dim,heads,dtype,kind", [
    (65, 256, 4, F32, I8), (129, 64, 3, BF16, E4M3), (200, 128, 5, F16, I8), (260, 256, 3, F32, E4M3),
    (400, 256, 1, BF16, I8), (513, 64, 9, F32, I8), (600, 128, 2, F32, E4M3), (1100, 256, 1, F16, E4M3),
])
def test_append_of_a_step_of_many_sequences(cuda, n, dim, heads, dtype, kind):
    """Blocks that get one token: growing, beginning anew, with infinities and NaN, unaligned rows."""
    from qwowl35_amd import attention as at

    c = _blocks(cuda, n + 1, heads, 64, dim, kind)
    want = blk.decode(c)
    randn = _gen(cuda, n)
    for step in range(3):
        slots = _steps(n, step)
        k = (randn(n, heads, dim + 1) * 6.0 ** step).to(dtype)[..., 1:]
        v = (randn(heads, n, dim) * 4.0 ** step).to(dtype).transpose(0, 1)
        k[20, 0, 3], k[21, heads - 1, 0], v[22, 0, dim - 1], v[24] = math.inf, math.nan, -math.inf, 0.0
        at.kv_append(c, k, v, slots.to(cuda))
        for state, x in zip(want, (k, v)):
            blk.append(state, x.double().cpu(), slots, kind)
        blk.same(c, want, f"step {step}")


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("dim,rot,sections,normed", [(256, 64, [11, 11, 10], True), (64, 64, [], False), (128, 128, [], True)])
def test_a_step_of_many_is_what_steps_of_few_make(cuda, kind, dim, rot, sections, normed):
    """The keys' rotation and norm, bit for bit, whichever way the step is cut into calls; and in a graph."""
    from qwowl35_amd import attention as at

    n, heads = 333, 3
    randn = _gen(cuda, dim)
    k, v = randn(n, heads, dim), randn(n, heads, dim)
    norm = randn(dim).abs() + 0.5 if normed else None
    rope = at.Rotary(rot, 1e7, sections, True, device=cuda)
    pos = torch.randint(0, 100000, (rope.axes, n), device=cuda, dtype=torch.int32)
    pos = pos if rope.axes > 1 else pos[0]
    i = torch.arange(n, device=cuda)
    slots = i * 32 + (i * 5) % 32
    few, many, graphed = (_blocks(cuda, n, heads, 32, dim, kind) for _ in range(3))
    for a in range(0, n, 37):
        at.kv_append(few, k[a:a + 37], v[a:a + 37], slots[a:a + 37], rope=rope,
                     positions=pos[..., a:a + 37].contiguous(), norm=norm)
    at.kv_append(many, k, v, slots, rope=rope, positions=pos, norm=norm)
    start = [x.clone() for x in (graphed.k.view(torch.uint8), graphed.v.view(torch.uint8), graphed.k_scale, graphed.v_scale)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        at.kv_append(graphed, k, v, slots, rope=rope, positions=pos, norm=norm)
    for _ in range(3):
        for x, was in zip((graphed.k.view(torch.uint8), graphed.v.view(torch.uint8), graphed.k_scale, graphed.v_scale), start):
            x.copy_(was)
        g.replay()
        torch.cuda.synchronize()
        for c in (many, graphed):
            for x, y in ((c.k, few.k), (c.v, few.v)):
                assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
            assert torch.equal(c.k_scale, few.k_scale) and torch.equal(c.v_scale, few.v_scale)


@pytest.mark.parametrize("dtype,kind", [(F32, I8), (BF16, E4M3)])
def test_append_of_unaligned_rows(cuda, dtype, kind):
    """Rows at odd element offsets, heads first, and no token at all."""
    from qwowl35_amd import attention as at

    c = _blocks(cuda, 3, 2, 64, 128, kind)
    want = blk.decode(c)
    randn = _gen(cuda, 6)
    slots = torch.arange(70) + 20
    k, v = randn(70, 2, 129).to(dtype)[..., 1:], randn(2, 70, 131).to(dtype).transpose(0, 1)[..., 2:130]
    at.kv_append(c, k, v, slots.to(cuda))
    for state, x in zip(want, (k, v)):
        blk.append(state, x.double().cpu(), slots, kind)
    blk.same(c, want)
    at.kv_append(c, k[:0], v[:0], slots[:0].to(cuda))
    at.kv_append(c, k[:3], v[:3], torch.tensor([-1, 192, -7], device=cuda))
    blk.same(c, want, "nothing to write")


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("dim,rot,sections,normed", [(256, 64, [11, 11, 10], True), (64, 64, [], False), (128, 32, [], True)])
def test_append_of_rotated_keys(cuda, kind, dim, rot, sections, normed):
    """Within half a step of the exact rotated key, beside the rotation's own fp32."""
    from qwowl35_amd import attention as at

    n, heads, page = 77, 2, 32
    c = _blocks(cuda, 5, heads, page, dim, kind)
    randn = _gen(cuda, dim)
    k, v = randn(n, heads, dim), randn(n, heads, dim)
    norm = randn(dim).abs() + 0.5 if normed else None
    rope = at.Rotary(rot, 1e7, sections, True, device=cuda)
    pos = torch.randint(0, 100000, (rope.axes, n), device=cuda, dtype=torch.int32)
    slots = torch.arange(n, device=cuda) + 32
    at.kv_append(c, k, v, slots, rope=rope, positions=pos if rope.axes > 1 else pos[0], norm=norm)
    want, bound = ref.rotate(k, rot, 1e7, pos if rope.axes > 1 else pos[0], sections, True, norm)
    codes, scales = blk.decode(c)[0]
    s = slots.cpu() // 32
    scale = scales[s, :, 0][..., None]
    got = codes[s, :, 0, slots.cpu() % 32] * scale
    step = scale / 2 if kind == I8 else torch.maximum(want.abs() * ref.EPS[E4M3], scale * ref.TINY[E4M3])
    assert ((got - want).abs() <= step + 2 * bound).all()
    for b in range(3):
        rows = slice(32 * b, min(32 * b + 32, n))
        m, off = want[rows].abs().amax((0, 2)), bound[rows].amax((0, 2))
        assert ((scales[b + 1, :, 0] == blk.fitting(m - off, kind)) | (scales[b + 1, :, 0] == blk.fitting(m + off, kind))).all()
    # (the last block's tokens behind the call are zero: it began anew)
    assert not codes[3, :, 0, n % 32:].any()


@pytest.mark.parametrize("kind", [I8, E4M3])
def test_special_numbers(cuda, kind):
    """Infinities, NaN, zeros, the largest and the smallest numbers; no block reaches another."""
    from qwowl35_amd import attention as at

    c = _blocks(cuda, 12, 1, 32, 64, kind)
    want = blk.decode(c)
    x = torch.zeros(12, 1, 64, device=cuda)
    x[0, 0, :4] = torch.tensor([math.inf, -math.inf, math.nan, 3.0])
    x[1, 0, :2] = torch.tensor([math.inf, math.nan])      # nothing finite but zeros
    x[3, 0, :3] = torch.tensor([3.4e38, -3.4e38, 1.0])
    x[4, 0, :3] = torch.tensor([1e-30, -1e-45, 2.0 ** -61])
    x[5, 0, 0] = 127.0 if kind == I8 else 448.0          # the largest code itself
    x[6, 0, 0] = torch.nextafter(torch.tensor(blk.TOP[kind]), torch.tensor(1e9))
    x[7, 0, :4] = torch.tensor([0.5, 1.5, 2.5, 100.0])   # ties
    x[8, 0, 0] = 2.0 ** -60
    x[9] = math.nan
    slots = torch.arange(12) * 32
    at.kv_append(c, x, x, slots.to(cuda))
    for state in want:
        blk.append(state, x.double().cpu(), slots, kind)
    blk.same(c, want)
    # a block of zeros grows from its first number on
    y = torch.full((1, 1, 64), 0.01, device=cuda)
    at.kv_append(c, y, y, torch.tensor([2 * 32 + 1], device=cuda))
    for state in want:
        blk.append(state, y.double().cpu(), [65], kind)
    blk.same(c, want)
    k, _ = at.kv_read(c, torch.tensor([65], device=cuda), dtype=F32)
    assert (k - 0.01).abs().max() <= 0.01 * 2.0 ** -4


@pytest.mark.parametrize("kind,most", [(I8, 1.0), (E4M3, 0.5)])
def test_growing_blocks_stay_near(cuda, kind, most):
    """Tokens ever larger: what the first ones have lost is less than a step of the last scale (half a step of their
    own and of the least code where codes are floating point)."""
    from qwowl35_amd import attention as at

    c = at.PagedCache.empty(1, 2, 32, 64, kind, device=cuda, block_scales=True)
    x = _gen(cuda, 4)(32, 2, 64) * torch.exp2(torch.arange(32, device=cuda) / 4.0)[:, None, None]
    for t in range(32):
        at.kv_append(c, x[t:t + 1], x[t:t + 1], torch.tensor([t], device=cuda))
    for (codes, scales), got in zip(blk.decode(c), at.kv_read(c, torch.arange(32, device=cuda), dtype=F32)):
        m = x.abs().amax((0, 2)).double().cpu()
        assert torch.equal(scales[0, :, 0], blk.fitting(m, kind))
        off = (got - x).abs().double().cpu()
        step = scales[0, :, 0][:, None]
        limit = most * step if kind == I8 else torch.maximum(2 ** -4 * x.abs().double().cpu(), 2 * step * 2.0 ** -10)
        assert (off <= limit).all()


def test_other_scales_double(cuda):
    """A block whose scale is no power of two (another quantiser's) keeps it, times powers of two."""
    from qwowl35_amd import attention as at

    c = _blocks(cuda, 1, 1, 32, 64, I8)
    c.k_scale.fill_(0.0123)
    c.v_scale.fill_(0.7)
    held = blk.decode(c)
    x = torch.full((1, 1, 64), 5.0, device=cuda)
    at.kv_append(c, x, x, torch.tensor([9], device=cuda))
    (kc, ks), (vc, vs) = blk.decode(c)
    s = float(torch.tensor(0.0123))
    assert float(ks) == 4 * s and float(vs) == float(torch.tensor(0.7))
    assert (kc[..., 9, :] == round(5.0 / (4 * s))).all() and (vc[..., 9, :] == 7).all()
    rest = [t for t in range(32) if t != 9]
    assert torch.equal(kc[..., rest, :], torch.round(held[0][0][..., rest, :] / 4))
    assert torch.equal(vc[..., rest, :], held[1][0][..., rest, :])


@pytest.mark.parametrize("kind", [I8, E4M3])
def test_past_four_gib(cuda, kind):
    """Slots whose byte offset passes 32 bits, at either end of the cache: written, read, attended over."""
    from qwowl35_amd import attention as at

    heads, page, dim = 8, 4096, 256
    pages = (1 << 32) // (heads * page * dim) + 3
    c = at.PagedCache.empty(pages, heads, page, dim, kind, device=cuda, block_scales=True)
    last = (pages - 1) * page
    slots = torch.tensor([0, pages * page - 32] + list(range(last, last + 40)), device=cuda)
    x = _gen(cuda, 3)(42, heads, dim)
    at.kv_append(c, x, -x, slots)
    k, v = at.kv_read(c, slots, dtype=F32)
    # half a step of the largest scale that a block of such tokens gets, of either type
    limit = torch.maximum(x.abs() * 2.0 ** -4, torch.tensor(2.0 ** -5 if kind == I8 else 2.0 ** -16, device=cuda))
    assert ((k - x).abs() <= limit).all() and ((v + x).abs() <= limit).all()
    table = torch.tensor([[pages - 1]], dtype=torch.int32, device=cuda)
    q = _gen(cuda, 4)(1, heads, dim).to(F16)
    got = at.prefix_attention(q, c, table, torch.tensor([40], dtype=torch.int32, device=cuda))
    want, bound = ref.attend(q, k[2:], v[2:], torch.ones(1, 40, dtype=torch.bool), dim ** -0.5, F16)
    ref.close(got, want, bound * (1 + 2.0 ** -5), "attention")


# ---- kv_read -------------------------------------------------------------------------------------------------------

READS = {
    "one": lambda page: [page + 5],
    "blocks": lambda page: list(range(page - 32, page + 64)),
    "ragged": lambda page: list(range(3, 50)),
    "order": lambda page: [9, 40, 8, 10, 9, 11, 2 * page + 31, 39, 0, 2 * page, 64 % page, 17],
    "outside": lambda page: [-1, 0, 1, 2, 10 ** 12, 3, 4, 3 * page, 5, -(2 ** 62)],
    "sparse": lambda page: list(range(0, 3 * page, 7)),
}


@pytest.mark.parametrize("slots", READS)
@pytest.mark.parametrize("dim,heads,page", [(64, 3, 64), (128, 1, 96), (256, 4, 64)])
@pytest.mark.parametrize("kind,blocks", [(I8, True), (E4M3, True), (E4M3, False), (F16, False), (BF16, False)])
@pytest.mark.parametrize("out", [F32, F16, BF16])
def test_read(cuda, slots, dim, heads, page, kind, blocks, out):
    """Bit for bit: element times scale in fp32, rounded once."""
    from qwowl35_amd import attention as at

    if blocks:
        c = _blocks(cuda, 3, heads, page, dim, kind, seed=dim)
        c.k_scale.mul_(1.37)  # (any scale)
    else:
        c = _cache(cuda, 3, heads, page, dim, kind)
        every = torch.arange(3 * page, device=cuda)
        randn = _gen(cuda, 9)
        ref.pack(c, every, randn(3 * page, heads, dim), randn(3 * page, heads, dim))
    where = torch.tensor(READS[slots](page), device=cuda)
    n = where.numel()
    live = (where >= 0) & (where < 3 * page)
    at_ = torch.where(live, where, 0)
    want = []
    for x, scale in zip(ref.unpack(c, at_), (c.k_scale, c.v_scale)):
        x = x.to(cuda).float()
        if blocks:
            x = x * scale[at_ // page, :, at_ % page // 32][..., None]
        elif scale is not None:
            x = x * scale[:, None]
        want.append(torch.where(live[:, None, None], x, 0.0).to(out))
    for got, w in zip(at.kv_read(c, where, dtype=out), want):
        assert got.dtype == out and torch.equal(got, w)
    # into rows that do not begin 16-byte aligned, heads first, and nothing beside them
    k = torch.full((n, heads, dim + 1), 7.0, dtype=out, device=cuda)
    v = torch.full((heads, n, dim), 7.0, dtype=out, device=cuda)
    rk, rv = at.kv_read(c, where, k=k[..., 1:], v=v.transpose(0, 1))
    assert torch.equal(rk, want[0]) and torch.equal(rv, want[1]) and (k[..., 0] == 7).all()


def test_read_refuses(cuda):
    from qwowl35_amd import Qw35Error
    from qwowl35_amd import attention as at

    c = _blocks(cuda, 2, 2, 32, 64, I8)
    where = torch.arange(3, device=cuda)
    for kw, what in (({"dtype": torch.int32}, "fp32, bf16 or fp16"), ({"k": torch.zeros(3, 2, 32, device=cuda)}, "k must be"),
                     ({"k": torch.zeros(3, 2, 64, device=cuda), "dtype": F16}, "k must be"),
                     ({"v": torch.zeros(3, 2, 64)}, "v must be"),
                     ({"k": torch.zeros(3, 2, 128, device=cuda)[..., ::2]}, "unit column stride")):
        with pytest.raises(Qw35Error, match=what):
            at.kv_read(c, where, **kw)
    for slots in (where.int(), where.cpu(), where[::2], where.view(1, 3)):
        with pytest.raises(Qw35Error, match="slots must be"):
            at.kv_read(c, slots)
    k, v = at.kv_read(c, where[:0])
    assert k.shape == v.shape == (0, 2, 64) and k.dtype == F16


def test_caches_refused(cuda):
    from qwowl35_amd import Qw35Error
    from qwowl35_amd import attention as at

    c = _blocks(cuda, 2, 2, 64, 64, I8)
    for args, what in (((c.k, c.v), "needs k_scale and v_scale"), ((c.k, c.v, c.k_scale), "needs k_scale and v_scale"),
                       ((c.k, c.v, c.k_scale, c.v_scale[..., :1]), "v_scale must be"),
                       ((c.k, c.v, c.k_scale.double(), c.v_scale), "k_scale must be"),
                       ((c.k, c.v, c.k_scale, c.v_scale.cpu()), "v_scale must be"),
                       ((c.k.half(), c.v.half(), c.k_scale, c.v_scale), "a cache is"),
                       ((c.k.view(torch.uint8), c.v.view(torch.uint8)), "a cache is")):
        with pytest.raises(Qw35Error, match=what):
            at.PagedCache(*args)
    with pytest.raises(Qw35Error, match="makes its own scales"):
        at.PagedCache.empty(2, 2, 64, 64, I8, device=cuda, k_scale=c.k_scale)
    with pytest.raises(Qw35Error, match="a cache is"):
        at.PagedCache.empty(2, 2, 64, 64, F16, device=cuda, block_scales=True)


def test_a_new_cache_holds_zeros(cuda):
    from qwowl35_amd import attention as at

    torch.empty(1 << 20, dtype=torch.uint8, device=cuda).fill_(0x7f)  # (memory that the caches may be given)
    for kind in (I8, E4M3):
        c = at.PagedCache.empty(2, 2, 64, 64, kind, device=cuda, block_scales=True)
        k, v = at.kv_read(c, torch.arange(128, device=cuda))
        assert bool((k == 0).all()) and bool((v == 0).all()) and c.block_scales

"""Rotary positions, the paged cache's append and shared-prefix attention
against their formulas in float64, at the sizes and masks where they can go
wrong, with bounds counted from the kernels' roundings."""
from __future__ import annotations

import math

import pytest
import torch

from tests import attention_reference as ref

pytestmark = pytest.mark.gpu

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn


def _gen(cuda, seed):
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    return lambda *shape: torch.randn(shape, generator=g, device=cuda)


# ---- rotate --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("n,heads,dim,rot,sections,interleaved", [
    (1, 16, 256, 64, [11, 11, 10], True),
    (7, 3, 128, 128, [16, 24, 24], False),
    (33, 1, 64, 32, [], False),
    (5, 2, 96, 48, [9, 8, 7], True),
    (2, 5, 8, 0, [], False),
    (3, 2, 512, 512, [100, 50, 50, 56], False),
    (4, 2, 256, 16, [3, 3, 2], True),
])
@pytest.mark.parametrize("dtype,out", [(F32, F16), (F32, F32), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("normed", [False, True])
def test_rotate(cuda, n, heads, dim, rot, sections, interleaved, dtype, out, normed):
    from qwowl35_amd import attention as at

    randn = _gen(cuda, n * dim + rot)
    x = randn(n, heads, 2 * dim).to(dtype)[..., :dim]  # (a gated projection's queries)
    norm = randn(dim).abs() + 0.5 if normed else None
    rope = at.Rotary(rot, 1e7, sections, interleaved, device=cuda) if rot else None
    axes = rope.axes if rope else 1
    pos = torch.randint(0, 1 << 18, (axes, n), device=cuda, dtype=torch.int32)
    pos[:, 0] = 0
    got = at.rotate(x, rope, pos if axes > 1 else pos[0], norm=norm, out_dtype=out)
    want, bound = ref.rotate(x, rot, 1e7, pos if axes > 1 else pos[0], sections, interleaved, norm)
    assert got.dtype == out and got.shape == x.shape
    ref.close(got, want, bound, "rotate")


def test_rotate_far_and_negative_positions(cuda):
    """Angles of positions up to 2^31: exact where fp32 (and float64's product) would lose them."""
    from qwowl35_amd import attention as at

    x = _gen(cuda, 3)(6, 2, 64)
    pos = torch.tensor([2 ** 31 - 1, -(2 ** 31), 2 ** 30 + 12345, -1, 262143, 1], device=cuda, dtype=torch.int32)
    got = at.rotate(x, at.Rotary(64, 10000.0, device=cuda), pos)
    want, bound = ref.rotate(x, 64, 10000.0, pos)
    # (the float64 reference's own angle is off by up to 2^31 2^-53 radians)
    ref.close(got, want, bound + want.abs().amax() * 2.0 ** -21, "far positions")


def test_rotate_in_place_unaligned_and_empty(cuda):
    from qwowl35_amd import attention as at

    randn = _gen(cuda, 5)
    rope = at.Rotary(32, 1e6, device=cuda)
    pos = torch.arange(9, device=cuda, dtype=torch.int32)
    base = randn(9 * 3 * 67 + 1)
    x = base[1:].view(9, 3, 67)[..., :64]  # rows at odd element offsets
    want, bound = ref.rotate(x, 32, 1e6, pos)
    out = torch.zeros(9, 3, 65, device=cuda)[..., 1:]
    ref.close(at.rotate(x, rope, pos, out=out), want, bound, "unaligned")
    edge = base.clone()
    at.rotate(x, rope, pos, out=x)
    ref.close(x, want, bound, "in place")
    assert torch.equal(base[1:].view(9, 3, 67)[..., 64:], edge[1:].view(9, 3, 67)[..., 64:])
    t = randn(3, 9, 64).transpose(0, 1)  # head-major storage
    want, bound = ref.rotate(t, 32, 1e6, pos)
    ref.close(at.rotate(t, rope, pos), want, bound, "head-major")
    assert at.rotate(x[:0], rope, pos[:0]).shape == (0, 3, 64)


def test_rotate_keeps_rows_apart(cuda):
    """A NaN in one row reaches no other; a zero row stays zero under the norm."""
    from qwowl35_amd import attention as at

    x = _gen(cuda, 6)(8, 4, 64)
    x[3, 2, 5] = math.nan
    x[4, 1] = 0
    pos = torch.arange(8, device=cuda, dtype=torch.int32)
    got = at.rotate(x, at.Rotary(64, 1e4, device=cuda), pos, norm=torch.ones(64, device=cuda))
    bad = torch.isnan(got).any(-1)
    assert bad[3, 2] and int(bad.sum()) == 1 and not got[4, 1].any()


# ---- kv_append -----------------------------------------------------------------------------------------------------

def _cache(cuda, pages, heads, page, dim, dtype, seed=1, scales=True):
    from qwowl35_amd import attention as at

    s = {}
    if dtype == E4M3 and scales:
        g = torch.Generator(device=cuda)
        g.manual_seed(seed)
        s = {k: torch.rand(heads, generator=g, device=cuda) * 0.02 + 0.005 for k in ("k_scale", "v_scale")}
    c = at.PagedCache.empty(pages, heads, page, dim, dtype, device=cuda, **s)
    c.k.view(torch.uint8).fill_(0x7f)  # NaN in each of the types
    c.v.view(torch.uint8).fill_(0x7f)
    return c


SLOTS = {
    "one": lambda page: [page + 5],
    "octets": lambda page: list(range(page - 8, page + 24)),         # whole granules, over a page's end
    "ragged": lambda page: list(range(3, 30)),                         # begins and ends inside granules
    "order": lambda page: [9, 8, 10, 11, 12, 13, 14, 15, 40, 17, 2 * page + 31, 16],
    "padding": lambda page: [-1, 0, 1, 2, -1, 3, 4, 10 ** 12, 5, 6, 7, 3 * page],
    "gap": lambda page: [0, 1, 2, 3, 4, 5, 6, 32 + 7],
}


@pytest.mark.parametrize("slots", SLOTS)
@pytest.mark.parametrize("dim,heads,page", [(64, 3, 32), (128, 1, 96), (256, 4, 64)])
@pytest.mark.parametrize("dtype,cache", [(F32, F16), (BF16, BF16), (F32, E4M3), (F16, E4M3)])
def test_kv_append(cuda, slots, dim, heads, page, dtype, cache):
    from qwowl35_amd import attention as at

    c = _cache(cuda, 3, heads, page, dim, cache)
    before = c.k.view(torch.uint8).clone(), c.v.view(torch.uint8).clone()
    where = torch.tensor(SLOTS[slots](page), dtype=torch.int64, device=cuda)
    n = where.numel()
    randn = _gen(cuda, dim + n)
    k, v = randn(n, heads, dim + 8).to(dtype)[..., :dim], randn(heads, n, dim).to(dtype).transpose(0, 1)
    norm = randn(dim).abs() + 0.5
    rope = at.Rotary(dim // 2, 1e7, [dim // 4 - 2 * (dim // 12), dim // 12, dim // 12], True, device=cuda)
    pos = torch.randint(0, 100000, (3, n), device=cuda, dtype=torch.int32)
    at.kv_append(c, k, v, where, rope=rope, positions=pos, norm=norm)
    live = ((where >= 0) & (where < 3 * page)).cpu()
    gk, gv = ref.unpack(c, where.cpu()[live])
    wk, bound = ref.rotate(k, dim // 2, 1e7, pos, rope.sections, True, norm)
    wv = v.double().cpu()
    if cache == E4M3:
        wk, bound = wk / c.k_scale.double().cpu()[:, None], bound / c.k_scale.double().cpu()[:, None]
        wv = wv / c.v_scale.double().cpu()[:, None]
        wk, wv = wk.clamp(-448, 448), wv.clamp(-448, 448)
    ref.close(gk, wk[live], (bound + wk.abs() * 2.0 ** -23)[live], "keys")
    ref.close(gv, wv[live], (wv.abs() * 2.0 ** -23)[live], "values")
    # nothing else was written: with the live slots' bytes put back, the pages are as before
    old = _cache(cuda, 3, heads, page, dim, cache)
    bk, bv = ref.unpack(old, where.cpu()[live])
    ref.pack(c, where.cpu()[live], bk, bv)
    assert torch.equal(c.k.view(torch.uint8), before[0]) and torch.equal(c.v.view(torch.uint8), before[1])


def test_kv_append_past_the_range_and_nan(cuda):
    from qwowl35_amd import attention as at

    c = _cache(cuda, 1, 1, 32, 64, E4M3, scales=False)
    v = torch.zeros(4, 1, 64, device=cuda)
    v[0], v[1], v[2], v[3] = 1e9, -1e9, math.nan, 2.0 ** -10  # (the last a tie of 0 and the least value: to even)
    at.kv_append(c, v, v, torch.arange(4, device=cuda))
    for got in ref.unpack(c, torch.arange(4)):
        got = got.float()
        assert (got[0] == 448).all() and (got[1] == -448).all() and got[2].isnan().all() and (got[3] == 0).all()
    c = _cache(cuda, 1, 1, 32, 64, F16)
    at.kv_append(c, v, v, torch.arange(4, device=cuda))
    k, _ = ref.unpack(c, torch.arange(4))
    assert k[0].isinf().all() and (k[0] > 0).all() and (k[1] < 0).all() and k[2].isnan().all()


def test_kv_append_past_four_gib(cuda):
    """Slots whose byte offset passes 32 bits, at either end of the cache."""
    from qwowl35_amd import attention as at

    heads, page, dim = 8, 4096, 256
    pages = (1 << 32) // (heads * page * dim) + 3
    c = at.PagedCache.empty(pages, heads, page, dim, E4M3, device=cuda)
    where = torch.tensor([0, pages * page - 1, (pages - 2) * page + 17], device=cuda)
    randn = _gen(cuda, 11)
    k, v = randn(3, heads, dim), randn(3, heads, dim)
    at.kv_append(c, k, v, where)
    gk, gv = ref.unpack(c, where)
    ref.close(gk, k.double().cpu(), 0.0 * k.double().cpu(), "keys")
    ref.close(gv, v.double().cpu(), 0.0 * v.double().cpu(), "values")
    table = torch.tensor([[pages - 1]], dtype=torch.int32, device=cuda)
    ref.pack(c, (pages - 1) * page + torch.arange(40), randn(40, heads, dim), randn(40, heads, dim))
    q = randn(1, heads, dim).to(F16)
    got = at.prefix_attention(q, c, table, torch.tensor([40], dtype=torch.int32, device=cuda))
    kk, vv = ref.unpack(c, (pages - 1) * page + torch.arange(40))
    want, bound = ref.attend(q, kk.float(), vv.float(), torch.ones(1, 40, dtype=torch.bool), dim ** -0.5, F16)
    ref.close(got, want, bound, "attention")


# ---- prefix_attention ----------------------------------------------------------------------------------------------

class Batch:
    """A batch over shuffled pages: NaN in every slot that no token fills."""

    def __init__(self, cuda, new, lens, prefix, heads, kv_heads, dim, page, dtype, cache, seed=0, more_pages=0,
                 spread=1.0):
        self.new, self.lens, self.prefix, self.dtype = new, lens, prefix, dtype
        count = lambda n: (n + page - 1) // page  # noqa: E731
        per = max([count(n) for n in lens] + [1]) + more_pages
        total = count(prefix) + sum(count(n) for n in lens) + 2
        self.cache = _cache(cuda, total, kv_heads, page, dim, cache, seed)
        randn = _gen(cuda, seed)
        order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        self.prefix_pages = order[:count(prefix)].to(cuda)
        table, at = torch.full((len(lens), per), -1, dtype=torch.int32), count(prefix)
        for s, n in enumerate(lens):
            table[s, :count(n)] = order[at:at + count(n)]
            at += count(n)
        self.pages = table.to(cuda)
        self.lengths = torch.tensor(lens, dtype=torch.int32, device=cuda)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        self.starts = torch.tensor(starts, dtype=torch.int32, device=cuda)
        self.q = (randn(starts[-1], heads, dim) * 2 * spread).to(dtype)
        size = 40.0 if cache == E4M3 else 1.0  # (times a scale of 0.005 .. 0.025)
        for pages, n in [(self.prefix_pages, prefix)] + [(self.pages[s], n) for s, n in enumerate(lens)]:
            if n:
                slots = self.cache.slots(pages, torch.arange(n, device=cuda))
                ref.pack(self.cache, slots, randn(n, kv_heads, dim) * size, randn(n, kv_heads, dim) * size)

    def tokens(self, s):
        """Keys and values of sequence s, prefix first, with their scales."""
        parts = []
        for pages, n in [(self.prefix_pages, self.prefix), (self.pages[s], self.lens[s])]:
            parts.append(ref.unpack(self.cache, self.cache.slots(pages, torch.arange(n, device=pages.device))))
        out = []
        for i, scale in enumerate((self.cache.k_scale, self.cache.v_scale)):
            t = torch.cat([p[i].float().double() for p in parts])
            out.append(t if scale is None else t * scale.double().cpu()[:, None])
        return out

    def want(self, window=0, sink=0, scale=None, gate=None):
        outs, bounds, first = [], [], 0
        for s, (new, length) in enumerate(zip(self.new, self.lens)):
            k, v = self.tokens(s)
            where = torch.arange(self.prefix + length)
            pos = self.prefix + length - new + torch.arange(new)[:, None]
            seen = where <= pos
            if window:
                seen = seen & ((where > pos - window) | (where < sink))
            o, b = ref.attend(self.q[first:first + new], k, v, seen, scale or self.q.shape[2] ** -0.5, self.dtype)
            outs.append(o)
            bounds.append(b)
            first += new
        o, b = torch.cat(outs), torch.cat(bounds)
        if gate is not None:
            g = torch.sigmoid(gate.double().cpu())
            o, b = o * g, b * g + (o * g).abs() * 2.0 ** -20  # (exp, sum and quotient of the gate)
        return o, b

    def run(self, **kw):
        from qwowl35_amd import attention as at

        kw = {"prefix_pages": self.prefix_pages, "prefix_len": self.prefix, "max_new": max(self.new), **kw}
        if "workspace" not in kw:  # (whatever it holds)
            kw["workspace"] = at.prefix_attention_workspace(self.cache, self.q.shape[1], len(self.lens),
                                                            self.q.shape[0])
            kw["workspace"].fill_(0xff)
        return at.prefix_attention(self.q, self.cache, self.pages, self.lengths, self.starts, **kw)


KINDS = [(F16, F16), (BF16, BF16), (F16, E4M3), (BF16, E4M3)]
SHAPES = {  # new, lens, prefix, heads, kv heads, page
    "one": ([1], [1], 0, 4, 1, 32),
    "tile_edges": ([1] * 5, [31, 32, 33, 64, 65], 0, 4, 2, 32),
    "empty": ([1, 1, 1], [0, 5, 0], 0, 2, 2, 32),                       # sequences that see nothing
    "prefix_only": ([1, 1], [0, 0], 37, 3, 1, 32),
    "prefix": ([1, 1, 1], [1, 40, 96], 100, 8, 2, 96),
    "no_new": ([0, 2, 0, 1], [9, 7, 0, 50], 33, 6, 2, 32),
    "rows_17": ([1] * 17, list(range(1, 18)), 70, 1, 1, 64),              # two 16-row tiles of the prefix
    "rows_60": ([3, 1, 4, 2], [30, 1, 64, 33], 129, 12, 2, 64),           # 60 rows, own tiles of mixed fill
    "chunk": ([70, 1, 9], [70, 33, 200], 65, 4, 1, 64),                   # causal within the chunk
    "chunk_long": ([40, 75], [300, 75], 0, 8, 4, 128),
    "late": ([5, 3], [2, 0], 0, 2, 1, 32),                                # more new tokens than lie in the cache
}


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype,cache", KINDS)
def test_prefix_attention(cuda, shape, dim, dtype, cache):
    new, lens, prefix, heads, kv_heads, page = SHAPES[shape]
    b = Batch(cuda, new, lens, prefix, heads, kv_heads, dim, page, dtype, cache, seed=len(shape) + dim)
    want, bound = b.want()
    got = b.run()
    assert got.dtype == dtype
    ref.close(got, want, bound, shape)
    ref.close(b.run(out_dtype=F32, max_new=0), want, bound, shape + " in fp32, rows divided for any sequence")


@pytest.mark.parametrize("window,sink", [(1, 0), (33, 0), (40, 5), (64, 64), (500, 3), (7, 400)])
@pytest.mark.parametrize("shape", ["prefix", "chunk", "rows_60", "tile_edges", "late"])
@pytest.mark.parametrize("dim,dtype,cache", [(64, BF16, BF16), (128, F16, E4M3), (256, F16, F16)])
def test_window_and_sink(cuda, window, sink, shape, dim, dtype, cache):
    new, lens, prefix, heads, kv_heads, page = SHAPES[shape]
    b = Batch(cuda, new, lens, prefix, heads, kv_heads, dim, page, dtype, cache, seed=window + dim)
    want, bound = b.want(window, sink)
    ref.close(b.run(window=window, sink=sink), want, bound, f"{shape} window {window} sink {sink}")


@pytest.mark.parametrize("gate", [F32, F16, BF16])
@pytest.mark.parametrize("shape", ["one", "prefix", "chunk"])
def test_gate_of_a_gated_projection(cuda, gate, shape):
    """The gate as the second half of each head's projection; a row that sees nothing stays zero."""
    new, lens, prefix, heads, kv_heads, page = SHAPES[shape]
    b = Batch(cuda, new, lens, prefix, heads, kv_heads, 128, page, F16, F16, seed=4)
    g = (_gen(cuda, 8)(b.q.shape[0], heads, 256) * 3).to(gate)[..., 128:]
    want, bound = b.want(gate=g)
    ref.close(b.run(gate=g), want, bound, "gate")
    ref.close(b.run(gate=g[:, :, ::1].contiguous()), want, bound, "contiguous gate")


@pytest.mark.parametrize("dim,dtype,cache", [(64, F16, F16), (256, BF16, E4M3)])
def test_many_pieces(cuda, dim, dtype, cache):
    """Lengths that are divided over the whole grid, of ragged sequences, and a workspace of a larger batch."""
    from qwowl35_amd import attention as at

    b = Batch(cuda, [1, 3, 1], [5000, 1, 777], 9000, 8, 2, dim, 64, dtype, cache, seed=2, more_pages=3)
    want, bound = b.want()
    ws = at.prefix_attention_workspace(b.cache, 8, 64, 300)
    first = b.run(workspace=ws)
    ref.close(first, want, bound, "many pieces")
    assert torch.equal(first, b.run(workspace=ws)), "the same call twice"


def test_peaked_rising_and_equal_scores(cuda):
    """Logits that rise along the sequence (the running maximum moves in every tile), one that outweighs all
    others, and keys that are all alike."""
    for kind in ("rising", "peak", "equal"):
        b = Batch(cuda, [1, 2], [200, 333], 0, 4, 2, 128, 32, F16, F16, seed=3)
        q0 = b.q[0, 0].float()
        unit = q0 / q0.norm()
        for s, n in enumerate(b.lens):
            slots = b.cache.slots(b.pages[s], torch.arange(n, device=cuda))
            _, v = ref.unpack(b.cache, slots)
            t = torch.arange(n, device=cuda, dtype=torch.float32)
            size = {"rising": t * 0.2, "peak": (t == n // 2) * 60.0, "equal": t * 0 + 1}[kind]
            ref.pack(b.cache, slots, (size[:, None] * unit)[:, None].expand(n, 2, 128), v)
        want, bound = b.want()
        ref.close(b.run(), want, bound, kind)


def test_infinities_and_nan_behind_the_mask(cuda):
    """Keys and values that a row does not see never reach it, whatever they are (later tokens of its chunk,
    tokens before its window); a row that sees a NaN has it."""
    for bad in (math.nan, math.inf):
        for dtype in (F16, BF16):
            b = Batch(cuda, [40], [70], 0, 4, 2, 64, 32, dtype, dtype, seed=5)
            slot = b.cache.slots(b.pages[0], torch.tensor([50], device=cuda))  # new token 20
            k, v = ref.unpack(b.cache, slot)
            v[0, :, 3] = bad
            k[0, :, 7] = math.nan if bad != bad else k[0, :, 7]
            clean, bound = b.want()
            ref.pack(b.cache, slot, k, v)
            got = b.run()
            ref.close(got[:20], clean[:20], bound[:20], "rows before")
            assert (got[20:, :, 3].isnan() | got[20:, :, 3].isinf()).all()
            if bad == bad:
                keep = [c for c in range(64) if c != 3]
                ref.close(got[20:, :, keep], clean[20:][..., keep], bound[20:][..., keep], "other columns")
            # out of every window: no row sees token 50 but the eight from it on
            want, bound = Batch.want(b, window=8)
            got = b.run(window=8)
            keep = [j for j in range(40) if j < 20 or j >= 28]
            ref.close(got[keep], want[keep], bound[keep], "outside the window")


def test_e4m3_nan_behind_the_mask(cuda):
    b = Batch(cuda, [9], [40], 0, 2, 1, 128, 32, F16, E4M3, seed=6)
    slot = b.cache.slots(b.pages[0], torch.tensor([36], device=cuda))  # new token 5
    k, v = ref.unpack(b.cache, slot)
    clean, bound = b.want()
    v = v.float()
    v[0, :, 100] = math.nan
    ref.pack(b.cache, slot, k.float(), v)
    got = b.run()
    ref.close(got[:5], clean[:5], bound[:5], "rows before")
    assert got[5:, :, 100].isnan().all() and not got[5:, :, :100].isnan().any()


def test_bad_device_data_stays_in_bounds(cuda):
    """Lengths past the table, page numbers outside the cache and starts past the tokens: what is there counts."""
    from qwowl35_amd import attention as at

    b = Batch(cuda, [1, 1, 1], [64, 96, 40], 0, 4, 2, 64, 32, F16, F16, seed=7)
    want, bound = b.want()
    pages, lengths = b.pages.clone(), b.lengths.clone()
    lengths[1] = 10 ** 9                     # the table holds 96
    pages[0, 1] = 10 ** 6                    # its second page is nowhere
    pages[2, 0] = -5
    got = at.prefix_attention(b.q, b.cache, pages, lengths, b.starts, max_new=1)
    ref.close(got[1:2], want[1:2], bound[1:2], "length past the table")
    k, v = b.tokens(0)
    o, bd = ref.attend(b.q[:1], k[:32], v[:32], torch.ones(1, 32, dtype=torch.bool), 64 ** -0.5, F16)
    ref.close(got[:1], o, bd, "a page outside the cache")
    k, v = b.tokens(2)
    o, bd = ref.attend(b.q[2:], k[32:], v[32:], torch.ones(1, 8, dtype=torch.bool), 64 ** -0.5, F16)
    ref.close(got[2:], o, bd, "the first page outside the cache")
    starts = torch.tensor([0, 1, 2, 900], dtype=torch.int32, device=cuda)
    ref.close(at.prefix_attention(b.q, b.cache, b.pages, b.lengths, starts), want, bound, "starts past the tokens")
    few = torch.tensor([0, 1, 2, 2], dtype=torch.int32, device=cuda)
    got = at.prefix_attention(b.q, b.cache, b.pages, b.lengths, few)
    ref.close(got[:2], want[:2], bound[:2], "tokens of no sequence")
    assert not got[2].any()
    negative = torch.tensor([-3, -1, -2], dtype=torch.int32, device=cuda)
    assert not at.prefix_attention(b.q, b.cache, b.pages, negative, b.starts).any()


def test_strides_of_queries_and_output(cuda):
    from qwowl35_amd import attention as at

    b = Batch(cuda, [2, 1], [40, 70], 50, 4, 2, 64, 32, F16, F16, seed=8)
    want, bound = b.want()
    odd = torch.empty(3 * 4 * 67 + 1, dtype=F16, device=cuda)[1:].view(3, 4, 67)[..., :64]
    odd.copy_(b.q)
    b.q = odd
    out = torch.zeros(3, 4, 65, dtype=F16, device=cuda)[..., 1:]
    ref.close(b.run(out=out), want, bound, "rows at odd offsets")
    b.q = odd.transpose(0, 1).contiguous().transpose(0, 1)
    base = torch.full((4, 3, 64), 7.0, dtype=F32, device=cuda)
    ref.close(b.run(out=base.transpose(0, 1)), want, bound, "head-major")
    starts, b.starts = b.starts, None
    b.new, b.lens = [1, 1, 1], [40, 70, 40]
    b.pages, b.lengths = b.pages[[0, 1, 0]].contiguous(), b.lengths[[0, 1, 0]].contiguous()
    want, bound = b.want()
    ref.close(b.run(), want, bound, "no starts: a token each")


def test_recorded_call_follows_the_lengths(cuda):
    """A captured append and attention replayed as the sequences grow, with eager work between the replays."""
    from qwowl35_amd import attention as at

    b = Batch(cuda, [1, 1], [20, 60], 40, 4, 2, 128, 32, F16, F16, seed=9, more_pages=2)
    b.pages[0, :3] = torch.tensor([b.pages[0, 0].item(), b.cache.n_pages - 1, 0], dtype=torch.int32)
    order = torch.randperm(12, generator=torch.Generator().manual_seed(1))  # a cache of its own, with room to grow
    big = _cache(cuda, 12, 2, 32, 128, F16)
    prefix = order[:2].to(torch.int32).to(cuda)
    pages = order[2:10].to(torch.int32).view(2, 4).to(cuda)
    randn = _gen(cuda, 10)
    kv = randn(2, 200, 2, 128)
    ref.pack(big, big.slots(prefix, torch.arange(40, device=cuda)), kv[0, :40], kv[1, :40])
    lengths = torch.tensor([0, 0], dtype=torch.int32, device=cuda)
    q = torch.empty(2, 4, 128, dtype=F16, device=cuda)
    k, v = torch.empty(2, 2, 128, device=cuda), torch.empty(2, 2, 128, device=cuda)
    slots, out = torch.empty(2, dtype=torch.int64, device=cuda), torch.empty(2, 4, 128, device=cuda)
    ws = at.prefix_attention_workspace(big, 4, 2, 2)

    def step():
        at.kv_append(big, k, v, slots)
        at.prefix_attention(q, big, pages, lengths, max_new=1, prefix_pages=prefix, prefix_len=40, out=out,
                            workspace=ws)

    side = torch.cuda.Stream()
    lengths.fill_(1)
    slots.fill_(-1)
    q.zero_()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    mine = [[], []]
    for i in range(70):
        lengths.copy_(torch.tensor([i + 1, max(0, i - 30)], dtype=torch.int32))
        new = [i, i - 31]
        slots.copy_(torch.stack([big.slots(pages[s], torch.tensor(n, device=cuda)) if n >= 0
                                 else torch.tensor(-1, device=cuda) for s, n in enumerate(new)]))
        k.copy_(randn(2, 2, 128))
        v.copy_(randn(2, 2, 128))
        q.copy_(randn(2, 4, 128))
        for s in range(2):
            if new[s] >= 0:
                mine[s].append((k[s].to(F16).cpu(), v[s].to(F16).cpu()))
        graph.replay()
        if i in (0, 30, 31, 32, 33, 69):
            for s in range(2):
                t = [torch.cat([kv[j, :40].to(F16).cpu()] + [p[j][None] for p in mine[s]]) for j in range(2)]
                seen = torch.ones(1, t[0].shape[0], dtype=torch.bool)
                want, bound = ref.attend(q[s:s + 1], t[0], t[1], seen, 128 ** -0.5, F16)
                ref.close(out[s:s + 1], want, bound, f"replay {i}, sequence {s}")


def test_another_stream(cuda):
    """Calls on a side stream, by argument and as the current one."""
    b = Batch(cuda, [1, 2], [33, 64], 20, 4, 2, 64, 32, F16, F16, seed=12)
    want, bound = b.want()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    a = b.run(stream=side, out=torch.zeros_like(b.q))
    with torch.cuda.stream(side):
        c = b.run()
    torch.cuda.synchronize()
    ref.close(a, want, bound, "stream argument")
    ref.close(c, want, bound, "current stream")


def test_nothing_to_do(cuda):
    b = Batch(cuda, [1], [5], 0, 2, 1, 64, 32, F16, F16)
    b.q = b.q[:0]
    b.starts = torch.zeros(2, dtype=torch.int32, device=cuda)
    assert b.run(workspace=None).shape == (0, 2, 64)

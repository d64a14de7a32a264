"""Forms of the attention kernels that only long or large calls take."""
from __future__ import annotations

import math

import pytest
import torch

from tests import attention_reference as ref
from tests.test_gpu_attention import BF16, E4M3, F16, F32, Batch

pytestmark = pytest.mark.gpu


def test_as_many_sequences_as_the_list_holds(cuda):
    """1580 sequences of a token each: with starts their row tiles are counted by an upper bound, which is refused."""
    from qwowl35_amd import Qw35Error

    b = Batch(cuda, [1] * 1580, [1 + s % 37 for s in range(1580)], 40, 2, 1, 256, 32, F16, F16, seed=1)
    want, bound = b.want()
    with pytest.raises(Qw35Error, match="row tiles in a call"):
        b.run()
    b.starts = None
    ref.close(b.run(), want, bound, "a token each")


ROWS = {  # new tokens of the sequences (one head: a new token is a row), shared tokens
    "own_16": ([1], 0), "own_shared_20": ([20], 0), "own_shared_100": ([100], 0), "own_32": ([20] + [1] * 140, 0),
    "prefix_16": ([1], 32), "prefix_32": ([20], 32), "prefix_64": ([50], 32), "prefix_shared": ([100], 32),
}


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("dim,dtype,cache", [(64, F16, F16), (128, F16, E4M3), (256, F16, F16), (64, BF16, BF16)])
def test_small_weights_beside_a_large_one(cuda, rows, dim, dtype, cache):
    """One token with nearly all the weight and a value of zero, 31 of 2^-26 or 2^-27 each with a value of one: the
    result is theirs."""
    new, prefix = ROWS[rows]
    more = 0 if prefix else 32
    b = Batch(cuda, new, [n + more for n in new], prefix, 1, 1, dim, 32, dtype, cache, seed=2)
    b.q.fill_(8.0 / dim ** 0.5)  # (logits are 8 times a key's columns)
    if cache == E4M3:
        b.cache.k_scale.fill_(1.0), b.cache.v_scale.fill_(1.0)
    top = 2.25 if cache == E4M3 else 2.34
    for s, n in enumerate(b.lens):
        k = torch.full((prefix + n, 1, dim), -9.0, device=cuda)  # the new tokens' own weights are nothing
        k[:32], k[0] = 0.0, top
        v = torch.ones(prefix + n, 1, dim, device=cuda)
        v[0] = 0.0
        slots = torch.cat([b.cache.slots(b.prefix_pages, torch.arange(prefix, device=cuda)),
                           b.cache.slots(b.pages[s], torch.arange(n, device=cuda))])
        ref.pack(b.cache, slots, k, v)
    want, _ = b.want()
    assert 31 * 2.0 ** -28 < float(want.min()) <= float(want.max()) < 31 * 2.0 ** -25
    # weights: rounded to the type, in fp16's subnormals by half a step of those (2^-25) against a largest one of at
    # least 2^7; exponentials and rescalings to 2^-18, and twice the logits' error
    off = 8.0 * top * (dim + 4) * 2.0 ** -24
    bound = (ref.EPS[dtype] + 2.0 ** -18 + 2 * off) * want + (2.0 ** -32 * 32 if dtype == F16 else 0.0)
    ref.close(b.run(out_dtype=F32), want, bound, rows)


FAR = {  # new tokens, shared tokens, heads
    "one_tile": ([1], 0, 1), "parts_16": ([1, 2], 0, 2), "shared_20": ([20], 0, 1), "shared_100": ([100], 0, 1),
    "alone_16": ([1] * 300, 0, 8), "alone_32": ([20] * 300, 0, 8), "alone_shared": ([70] * 70, 0, 8),
    "prefix_16": ([1], 64, 1), "prefix_64": ([50], 64, 1), "prefix_shared": ([100], 64, 2),
}


@pytest.mark.parametrize("rows,dim", [(r, d) for r in FAR for d in (64, 128, 256) if d == 64 or FAR[r][2] < 8])
def test_an_infinity_of_small_weight_stays_one(cuda, rows, dim):
    """Weights of 2^-40, which fp16 rounds to zero: a value that is infinite is so in the result, NaN of both signs."""
    new, prefix, heads = FAR[rows]
    more = 0 if prefix else 31 if rows == "one_tile" else 40
    b = Batch(cuda, new, [n + more for n in new], prefix, heads, heads, dim, 32, F16, F16, seed=3)
    b.q.fill_(8.0 / dim ** 0.5)
    where = [(b.prefix_pages, prefix)] if prefix else list(zip(b.pages, b.lens))
    for pages, n in where:
        slots = b.cache.slots(pages, torch.arange(n, device=cuda))
        k, v = ref.unpack(b.cache, slots)
        k[:2], k[2:] = -27.7 / 8, k[2:].clamp(-0.02, 0.02)
        ref.pack(b.cache, slots, k, v)
    if prefix:  # (and the new tokens' own ones)
        for s, n in enumerate(b.lens):
            slots = b.cache.slots(b.pages[s], torch.arange(n, device=cuda))
            k, v = ref.unpack(b.cache, slots)
            ref.pack(b.cache, slots, k.clamp(-0.02, 0.02), v)
    clean, bound = b.want()
    for pages, _ in where:
        slots = b.cache.slots(pages, torch.arange(2, device=cuda))
        k, v = ref.unpack(b.cache, slots)
        v[0, :, 3], v[0, :, 5], v[1, :, 9] = math.inf, -math.inf, math.nan
        v[0, :, 7], v[1, :, 7] = math.inf, -math.inf
        v[0, :, dim - 1], v[1, :, dim - 1] = 1.0, -math.inf
        ref.pack(b.cache, slots, k, v)
    for out in (F16, F32):
        got = b.run(out_dtype=out)
        assert (got[..., 3] == math.inf).all() and (got[..., 5] == -math.inf).all()
        assert got[..., 7].isnan().all() and got[..., 9].isnan().all() and (got[..., dim - 1] == -math.inf).all()
        keep = [c for c in range(dim - 1) if c not in (3, 5, 7, 9)]
        ref.close(got[..., keep], clean[..., keep], bound[..., keep], rows)


@pytest.mark.parametrize("window,sink", [(100, 0), (100, 8), (40, 3)])
def test_an_infinity_outside_the_window_is_not_looked_at(cuda, window, sink):
    """A row whose result is lost to an infinity that it sees gets that one and none that it does not see."""
    b = Batch(cuda, [2], [300], 0, 1, 1, 64, 32, F16, F16, seed=4)
    b.q.fill_(1.0)
    slots = b.cache.slots(b.pages[0], torch.arange(300, device=cuda))
    k, v = ref.unpack(b.cache, slots)
    k[:], v[:] = 0.0, 1.0
    k[270] = -3.46
    v[270, :, 3] = math.inf                       # seen, of weight 2^-40
    v[150, :, 3], v[150, :, 4] = -math.inf, -math.inf  # before either window, behind the sinks
    if sink:
        k[1], v[1, :, 5] = -3.46, -math.inf
    ref.pack(b.cache, slots, k, v)
    got = b.run(window=window, sink=sink)
    assert (got[..., 3] == math.inf).all() and (got[..., 4] == 1.0).all()
    assert (got[..., 5] == (-math.inf if sink else 1.0)).all()


# ---- rows whose maximum rises --------------------------------------------------------------------------------------

RISING = {  # new tokens, shared tokens (of 64 columns; half of 256), tiles a wave or workgroup is from its last one
    "own_16": ([1] * 300, 0, 1), "own_32": ([20] * 300, 0, 1), "own_shared": ([70] * 70, 0, 1),
    "prefix_16": ([1], 24576, 4), "prefix_32": ([20], 24576, 4), "prefix_64": ([50], 24576, 2),
    "prefix_shared": ([100], 12288, 1), "prefix_abreast": ([300], 12288, 1),
}


def _dense(q, k, v, seen, scale, dtype):
    """(out, bound) of rows q [n, dim] over tokens k, v [t, dim], seen [n, t], in float64; v is not negative."""
    q, k, v = (t.double() for t in (q, k, v))
    s = (q @ k.t() * scale).masked_fill(~seen, -math.inf)
    out = torch.softmax(s, -1) @ v
    off = float((q.abs() @ k.abs().t()).max()) * abs(scale) * (q.shape[1] + 4) * 2.0 ** -24
    return out, (ref.EPS[dtype] + 2.0 ** -18 + 2 * off) * out


@pytest.mark.parametrize("rows", RISING)
@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16), (256, F16)])
def test_sums_follow_a_rising_maximum(cuda, rows, dim, dtype):
    """Every tile's scores are past the reference by more than its slack, and each column's result is the sum that one
    tile left before the later ones rescaled it (values elsewhere are zero)."""
    from qwowl35_amd import attention as at

    new, prefix, apart = RISING[rows]
    prefix = prefix // (2 if dim == 256 else 1)
    heads, page, n = 8, 64, sum(new)
    own = max(new) + (0 if prefix else 128)
    per, shared = (own + page - 1) // page, prefix // page
    cache = at.PagedCache.empty(shared + len(new) * per, heads, page, dim, dtype, device=cuda)
    pages = shared + torch.arange(len(new) * per, dtype=torch.int32, device=cuda).view(len(new), per)
    g = torch.Generator(device=cuda)
    g.manual_seed(6)
    randn = lambda *s: torch.randn(s, generator=g, device=cuda)  # noqa: E731
    q = (1 + 0.02 * randn(n, heads, dim)).to(dtype)
    many = prefix or 128
    tile = torch.arange(many, device=cuda) // 32
    rise = 18.0 / apart  # log2, of a tile
    k = (tile * (rise * math.log(2) * dim ** -0.5))[:, None, None] + 0.003 * randn(many, heads, dim)
    which = torch.arange(dim, device=cuda) % 8
    v = (tile[:, None] % 8 == which)[:, None] * (1 + 0.2 * randn(many, heads, dim)).clamp(0.5, 1.5)
    low = torch.full((max(new), heads, dim), -200.0 * dim ** -0.5, device=cuda)  # the new tokens: of no weight
    zero = torch.zeros_like(low)
    if prefix:
        ref.pack(cache, torch.arange(prefix, device=cuda), k, v)
        tokens = [(low, zero)] * len(new)
    else:
        tokens = [(torch.cat([k, low]), torch.cat([v, zero]))] * len(new)
    for s in range(len(new)):
        m = tokens[s][0].shape[0]
        ref.pack(cache, cache.slots(pages[s], torch.arange(m, device=cuda)), *tokens[s])
    lengths = torch.full((len(new),), own, dtype=torch.int32, device=cuda)
    starts = torch.arange(len(new) + 1, dtype=torch.int32, device=cuda) * new[0]
    got = at.prefix_attention(q, cache, pages, lengths, starts, max_new=max(new), out_dtype=F32, prefix_len=prefix,
                              prefix_pages=torch.arange(shared, dtype=torch.int32, device=cuda) if prefix else None)
    kk, vv = k.to(dtype).double(), v.to(dtype).double()
    for h in range(heads):
        want, bound = _dense(q[:, h], kk[:, h], vv[:, h], torch.ones(n, many, dtype=torch.bool, device=cuda), dim ** -0.5,
                             dtype)
        there = want > 2.0 ** -80
        assert there.any(0).sum() >= dim // 8 * 4
        ref.close(torch.where(there, got[:, h], 0.0), torch.where(there, want, 0.0).cpu(),
                  torch.where(there, bound, 0.0).cpu(), f"{rows}, head {h}")


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("dim,dtype,cache", [(64, F16, E4M3), (128, BF16, BF16), (256, F16, F16)])
def test_widely_spread_scores(cuda, rows, dim, dtype, cache):
    """Logits of deviation 16: maxima rise past the slack again and again."""
    new, prefix = ROWS[rows]
    b = Batch(cuda, new, [n + 200 for n in new], 10 * prefix, 1, 1, dim, 32, dtype, cache, seed=8, spread=8.0)
    want, bound = b.want()
    ref.close(b.run(), want, bound, rows)


# ---- long and large calls ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("n,heads,dim", [(13108, 13, 64), (5500, 6, 64), (3000, 7, 128), (1100, 31, 256)])
@pytest.mark.parametrize("dtype,out", [(F32, F16), (BF16, BF16)])
def test_rotate_of_long_prompts(cuda, n, heads, dim, dtype, out):
    """Four and eight heads a lane, of head counts that these do not divide."""
    from qwowl35_amd import attention as at

    g = torch.Generator(device=cuda)
    g.manual_seed(n)
    x = torch.randn(n, heads, dim, generator=g, device=cuda).to(dtype)
    norm = torch.rand(dim, generator=g, device=cuda) + 0.5
    pos = torch.randint(0, 1 << 18, (3, n), generator=g, device=cuda, dtype=torch.int32)
    rope = at.Rotary(32, 1e7, [6, 5, 5], True, device=cuda)
    got = at.rotate(x, rope, pos, norm=norm, out_dtype=out)
    want, bound = ref.rotate(x, 32, 1e7, pos, [6, 5, 5], True, norm)
    ref.close(got, want, bound, "rotate")


@pytest.mark.parametrize("n,heads,dim", [(5500, 6, 64), (2100, 9, 128)])
@pytest.mark.parametrize("dtype,cache", [(F32, F16), (BF16, E4M3)])
def test_append_of_long_prompts(cuda, n, heads, dim, dtype, cache):
    """Four heads a lane, of head counts that these do not divide; tokens in shuffled pages, one in nine left out."""
    from qwowl35_amd import attention as at
    from tests.test_gpu_attention import _cache

    page = 96
    pages = (n + page - 1) // page + 1
    c = _cache(cuda, pages, heads, page, dim, cache)
    g = torch.Generator(device=cuda)
    g.manual_seed(n)
    k, v = (torch.randn(n, heads, dim, generator=g, device=cuda).to(dtype) for _ in range(2))
    order = torch.randperm(pages, generator=g, device=cuda)
    t = torch.arange(n, device=cuda) + 40
    slots = order[t // page] * page + t % page
    slots[::9] = -1
    pos = torch.randint(0, 1 << 18, (n,), generator=g, device=cuda, dtype=torch.int32)
    at.kv_append(c, k, v, slots, at.Rotary(dim, 1e6, device=cuda), pos)
    live = (slots >= 0).cpu()
    gk, gv = ref.unpack(c, slots.cpu()[live])
    wk, bound = ref.rotate(k, dim, 1e6, pos)
    wv = v.double().cpu()
    if cache == E4M3:
        wk, bound = wk / c.k_scale.double().cpu()[:, None], bound / c.k_scale.double().cpu()[:, None]
        wk, wv = wk.clamp(-448, 448), (wv / c.v_scale.double().cpu()[:, None]).clamp(-448, 448)
    ref.close(gk, wk[live], (bound + wk.abs() * 2.0 ** -23)[live], "keys")
    ref.close(gv, wv[live], (wv.abs() * 2.0 ** -23)[live], "values")


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_more_rows_than_the_join_gives_four_waves(cuda, dim):
    """1040 rows and more: a wave of the join has a row."""
    b = Batch(cuda, [90, 1, 39], [300, 60, 39], 333, 8, 2, dim, 32, F16, F16, seed=9)
    want, bound = b.want()
    ref.close(b.run(), want, bound, "after a prefix")
    want, bound = b.want(window=100, sink=5)
    ref.close(b.run(window=100, sink=5), want, bound, "in a window")


def _long(cuda, tokens, heads, dim, dtype, seqs=1, seed=1):
    """A cache of random tokens, each sequence's pages in a row."""
    from qwowl35_amd import attention as at

    page = 256
    per = (tokens + page - 1) // page
    cache = at.PagedCache.empty(seqs * per, heads, page, dim, F16 if dtype == E4M3 else dtype, device=cuda)
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    cache.k.normal_(generator=g)
    cache.v.normal_(generator=g)
    if dtype == E4M3:
        cache = at.PagedCache(cache.k.to(E4M3), cache.v.to(E4M3))
    return cache, torch.arange(seqs * per, dtype=torch.int32, device=cuda).view(seqs, per), g


def _one(q, cache, slots, h, upto=None):
    """(out, bound) of rows q [n, dim] over all of the tokens in `slots` of kv head h, in float64; row j sees all but
    the last n - 1 - j of them if `upto`."""
    page, dim = cache.page_size, cache.head_dim
    pg, at = slots // page, slots % page
    byte = torch.uint8 if cache.k.dtype == E4M3 else cache.k.dtype
    k = cache.k.view(byte)[:, h].permute(0, 1, 3, 2, 4)[pg, at // 32, at % 32].reshape(-1, dim).view(cache.k.dtype).double()
    v = cache.v.view(byte)[:, h].permute(0, 1, 3, 2)[pg, at // 8, at % 8].contiguous().view(cache.k.dtype).double()
    n, t = q.shape[0], slots.numel()
    seen = torch.ones(n, t, dtype=torch.bool, device=q.device)
    if upto:
        seen &= torch.arange(t, device=q.device) <= t - n + torch.arange(n, device=q.device)[:, None]
    s = (q.double() @ k.t() * dim ** -0.5).masked_fill(~seen, -math.inf)
    p = torch.softmax(s, -1)
    off = float((q.double().abs() @ k.abs().t()).max()) * dim ** -0.5 * (dim + 4) * 2.0 ** -24
    tiny = 2.0 ** -32 if q.dtype == F16 else 0.0
    return (p @ v).cpu(), ((ref.EPS[q.dtype] + 2.0 ** -18 + 2 * off) * (p @ v.abs()) + tiny * t * v.abs().max()).cpu()


@pytest.mark.parametrize("dim,dtype,cache", [(256, F16, F16), (64, BF16, BF16), (128, F16, E4M3)])
@pytest.mark.parametrize("kind", ["plain", "rising", "falling"])
def test_more_parts_than_a_round_of_the_join(cuda, dim, dtype, cache, kind):
    """One row over 70000 tokens: up to 2048 parts, which the join takes 256 at a time, rescaling what it has."""
    c, pages, g = _long(cuda, 70000, 1, dim, cache)
    tokens = 70000
    if kind != "plain":  # logits that go from 0 to 30
        up = torch.linspace(0, 30, tokens, device=cuda) * dim ** -0.5
        k, v = torch.randn(tokens, 1, dim, generator=g, device=cuda), torch.randn(tokens, 1, dim, generator=g, device=cuda)
        k = (0.5 * k + (up if kind == "rising" else up.flip(0))[:, None, None]).to(c.k.dtype)
        ref.pack(c, torch.arange(tokens, device=cuda), k, v.to(c.k.dtype))
    q = (torch.ones(1, 1, dim, device=cuda) + 0.1 * torch.randn(1, 1, dim, generator=g, device=cuda)).to(dtype)
    from qwowl35_amd import attention as at

    got = at.prefix_attention(q, c, pages, torch.tensor([tokens], dtype=torch.int32, device=cuda), out_dtype=F32)
    want, bound = _one(q[:, 0], c, torch.arange(tokens, device=cuda), 0)
    ref.close(got[:, 0], want, bound, kind)


@pytest.mark.parametrize("form", ["own_16", "prefix_16", "prefix_shared", "own_shared"])
def test_more_tiles_of_a_wave_than_are_looked_up_at_once(cuda, form):
    """A wave's 65th tile and those after it."""
    from qwowl35_amd import attention as at

    heads, dim = 8, 64
    seqs, tokens, new, prefix = {"own_16": (70, 8448, 1, 0), "prefix_16": (1, 64, 1, 540672), "prefix_shared": (1, 600, 600, 35072),
                                 "own_shared": (70, 2304, 72, 0)}[form]
    c, pages, g = _long(cuda, (prefix + tokens) if prefix else tokens, heads, dim, F16, seqs)
    shared = pages[0, :prefix // 256] if prefix else None
    own = pages[:, prefix // 256:].contiguous()
    q = torch.randn(seqs * new, heads, dim, generator=g, device=cuda).to(F16)
    lengths = torch.full((seqs,), tokens, dtype=torch.int32, device=cuda)
    starts = torch.arange(seqs + 1, dtype=torch.int32, device=cuda) * new
    got = at.prefix_attention(q, c, own, lengths, starts, max_new=new, prefix_pages=shared, prefix_len=prefix, out_dtype=F32)
    for s, h in {(0, 0), (seqs // 2, 3), (seqs - 1, 7)}:
        slots = c.slots(own[s], torch.arange(tokens, device=cuda))
        if prefix:
            slots = torch.cat([c.slots(shared, torch.arange(prefix, device=cuda)), slots])
        want, bound = _one(q[s * new:(s + 1) * new, h], c, slots, h, upto=True)
        ref.close(got[s * new:(s + 1) * new, h], want, bound, f"sequence {s}, head {h}")


@pytest.mark.parametrize("new", [17, 32, 33, 64])
@pytest.mark.parametrize("dim,dtype,cache", [(64, F16, F16), (128, BF16, E4M3), (256, F16, F16)])
def test_some_rows_of_many_sequences(cuda, new, dim, dtype, cache):
    """17 to 64 rows where there are many units: each wave has 32 of them and its own tiles."""
    b = Batch(cuda, [1] * 140 + [new], [1 + s % 40 for s in range(140)] + [new + 90], 70, 1, 1, dim, 32, dtype, cache,
              seed=new)
    want, bound = b.want()
    ref.close(b.run(), want, bound, f"{new} rows")
    want, bound = b.want(window=30, sink=3)
    ref.close(b.run(window=30, sink=3), want, bound, f"{new} rows in a window")


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_infinities_that_some_rows_of_many_sequences_see(cuda, bad, dtype):
    b = Batch(cuda, [60] + [1] * 140, [70] + [5] * 140, 0, 1, 1, 64, 32, dtype, dtype, seed=16)
    slot = b.cache.slots(b.pages[0], torch.tensor([40], device=cuda))  # new token 30
    k, v = ref.unpack(b.cache, slot)
    clean, bound = b.want()
    v[0, :, 3] = bad
    ref.pack(b.cache, slot, k, v)
    got = b.run()
    ref.close(got[:30], clean[:30], bound[:30], "rows before")
    ref.close(got[60:], clean[60:], bound[60:], "other sequences")
    hit = got[30:60, :, 3].double().cpu()
    assert torch.isnan(hit).all() if math.isnan(bad) else (hit == bad).all()
    keep = [c for c in range(64) if c != 3]
    ref.close(got[30:60][..., keep], clean[30:60][..., keep], bound[30:60][..., keep], "other columns")


@pytest.mark.parametrize("seqs", [8, 9, 64, 65])
@pytest.mark.parametrize("new", [17, 33])
def test_either_side_of_few_units(cuda, seqs, new):
    """Two kv heads of 64 columns: 17 rows share their tiles up to 8 sequences, 33 up to 64."""
    from qwowl35_amd import attention as at

    b = Batch(cuda, [new] + [3] * (seqs - 1), [new + 300] + [3 + 7 * (s % 40) for s in range(seqs - 1)], 40, 2, 2, 64, 32,
              F16, F16, seed=seqs)
    want, bound = b.want()
    ws = at.prefix_attention_workspace(b.cache, 2, 80, 300)
    ref.close(b.run(workspace=ws), want, bound, f"{seqs} sequences")

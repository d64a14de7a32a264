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
    "own_16": ([1], 0), "own_shared_20": ([20], 0), "own_shared_100": ([100], 0), "own_32": ([20] + [1] * 70, 0),
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

"""Forms of the attention kernels that only long or large calls take."""
from __future__ import annotations

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

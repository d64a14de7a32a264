"""Infinities and NaN that are appended to a block-scaled cache, by the rules of the header."""
from __future__ import annotations

import math

import pytest
import torch

from tests import block_reference as blk
from tests.test_gpu_attention import E4M3, F32

pytestmark = pytest.mark.gpu

I8 = torch.int8


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("n", [1, 100])
def test_infinities_and_nan(cuda, kind, n):
    """The largest code beside a number or under the scale of one; nothing where the block has neither: its scale is
    zero then, and the next call begins it anew.  (n calls' worth of tokens elsewhere take the call other ways.)"""
    from qwowl35_amd import attention as at

    top = blk.TOP[kind]
    c = at.PagedCache.empty(n + 4, 1, 32, 64, kind, device=cuda, block_scales=True)
    x = torch.zeros(n + 4, 1, 64, device=cuda)
    x[4:] = 1.0
    x[0, 0, :4] = torch.tensor([math.inf, -math.inf, math.nan, 3.0])
    x[1, 0, :3] = torch.tensor([math.inf, -math.inf, math.nan])  # no number but zeros
    x[2, 0, 0] = 2.0
    slots = torch.arange(n + 4, device=cuda) * 32
    at.kv_append(c, x, -x, slots)
    x[2, 0, :2] = torch.tensor([0.0, math.inf])  # under the scale that the block has
    at.kv_append(c, x[2:3], -x[2:3], slots[2:3] + 1)
    s = 2.0 ** (-5 if kind == I8 else -7)        # 3 <= top s
    for (codes, scales), sign in zip(blk.decode(c), (1, -1)):
        assert scales[0, 0, 0] == s and scales[1, 0, 0] == 0 and scales[3, 0, 0] == 0
        first = codes[0, 0, 0, 0]
        assert first[:2].tolist() == [sign * top, -sign * top] and first[3] == sign * 3.0 / s
        assert not codes[1, 0, 0, 0, :2].any() and not codes[1, 0, 0, 0, 3:].any()
        assert codes[2, 0, 0, 1, 1] == sign * top and scales[2, 0, 0] == (2.0 ** -5 if kind == I8 else 2.0 ** -7)
        for row in (first, codes[1, 0, 0, 0]):
            assert row[2] == 0 if kind == I8 else row[2].isnan()
    for got, sign in zip(at.kv_read(c, slots[:3], dtype=F32), (1, -1)):
        assert got[0, 0, :2].tolist() == [sign * top * s, -sign * top * s]
        assert not got[1, 0, :2].any() and bool(got[1, 0, 2].isnan()) == (kind == E4M3)
    y = torch.full((1, 1, 64), 0.5, device=cuda)
    at.kv_append(c, y, y, slots[1:2] + 7)
    for got in at.kv_read(c, slots[1:2] + torch.arange(32, device=cuda), dtype=F32):
        assert (got[7] == 0.5).all() and not got[:7].any() and not got[8:].any()

"""Attention over a block-scaled cache whose scales differ by whatever its format
allows: blocks of zero values, scales from one end of the range to the other."""
from __future__ import annotations

import pytest
import torch

from tests.block_reference import BLOCK, BlockBatch, close
from tests.test_gpu_attention import BF16, E4M3, F16, F32, SHAPES

pytestmark = pytest.mark.gpu

I8 = torch.int8
KINDS = [(F16, I8), (F16, E4M3), (BF16, E4M3)]

LONG = {  # new, lens, prefix, heads, kv heads, page
    "pieces": ([1, 3, 1], [3000, 1, 777], 5000, 8, 2, 64),                    # over the whole grid
    "shared": ([200], [900], 1500, 4, 2, 96),                                 # tiles that four waves share
    "many": ([1] * 260, [350 + s % 90 for s in range(260)], 0, 2, 2, 32),     # a wave has several tiles of a unit
}
PATHS = [(64, "many"), (64, "shared"), (128, "prefix"), (128, "chunk_long"), (128, "pieces"), (128, "shared"),
         (256, "many"), (256, "rows_60"), (256, "shared")]


def _batch(cuda, shape, dim, dtype, kind, seed, **kw):
    new, lens, prefix, heads, kv_heads, page = (SHAPES | LONG)[shape]
    return BlockBatch(cuda, new, lens, prefix, heads, kv_heads, dim, page, dtype, kind, seed=seed, **kw)


def _order(b):
    """The cache's blocks in the order of the tokens, [page, block of the page] of each, prefix and sequences apart."""
    per = b.cache.page_size // BLOCK
    for pages, n in [(b.prefix_pages, b.prefix)] + [(b.pages[s], n) for s, n in enumerate(b.lens)]:
        at = torch.arange((n + BLOCK - 1) // BLOCK, device=pages.device)
        if n:
            yield pages[at // per].long(), at % per


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("dim,shape", PATHS)
@pytest.mark.parametrize("less", [12, 24, 33, 50])
def test_blocks_of_zero_values_beside_small_ones(cuda, dtype, kind, dim, shape, less):
    """Blocks of zero values first in each sequence and here and there, the others' 2^-less of the usual and their
    logits lower: what a row gets is what the others weigh.  (The bound is relative to that.)"""
    b = _batch(cuda, shape, dim, dtype, kind, seed=less)
    b.cache.v_scale.mul_(2.0 ** -less)
    g = torch.Generator().manual_seed(less)
    for page, at in _order(b):
        zero = torch.rand(len(page), generator=g) < 0.3
        zero[0] = True
        zero = zero.to(cuda)
        b.cache.v_scale[page[zero], :, at[zero]] = 0.0
        b.cache.k_scale[page[zero], :, at[zero]] *= 2.0
    want, bound = b.want()
    close(b.run(out_dtype=F32), want, bound, f"{shape}, the others 2^-{less}")

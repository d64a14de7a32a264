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
    b = BlockBatch(cuda, new, lens, prefix, heads, kv_heads, dim, page, dtype, kind, seed=seed, **kw)
    if kind == E4M3:  # (no code past 448, which is NaN: rows that are numbers)
        for codes, scale in ((b.cache.k, b.cache.k_scale), (b.cache.v, b.cache.v_scale)):
            held = ~scale.isnan()[..., None].expand(-1, -1, -1, codes[0, 0].numel() // scale.shape[2]).reshape(codes.shape)
            codes.copy_(codes.float().masked_fill_(codes.isnan() & held, 416.0))
    return b


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


APART = {  # log2 of the values' scale of block i of n of a sequence, and how much higher its logits' spread is
    "any": lambda i, n, g: (torch.randint(-60, 113, (n,), generator=g), torch.ones(n)),
    "ends": lambda i, n, g: (torch.where(torch.rand(n, generator=g) < 0.5, -60, 112), torch.ones(n)),
    "small_first": lambda i, n, g: (torch.where(i <= n // 2, -60, 112), torch.ones(n)),
    "large_first": lambda i, n, g: (torch.where(i <= n // 2, 112, -60), torch.ones(n)),
    # small values at the softmax' large terms, so that either decides about a part of the result
    "small_louder": lambda i, n, g: ((e := torch.randint(-60, 113, (n,), generator=g)), torch.where(e < 20, 16.0, 1.0)),
    "zeros_too": lambda i, n, g: (torch.where(torch.rand(n, generator=g) < 0.3, -1000,
                                              torch.randint(-60, 113, (n,), generator=g)), torch.ones(n)),
}


def _wider(bound):
    """want()'s bound for scales so far apart.

    Six sums of exponents below 2^8 and the logarithm of a scale below 2^7 within two steps: 2^-14 of a row's sum of
    magnitudes, of which the bound has 2^-11 and more.

    And beside a row's largest value what fp32 does not hold (a column may have nothing else: codes of zero).  bf16
    weights under 2^-100 of the largest are dropped, and a part of a row counts 2^-123 at least, with sums of up to 2^33
    (the reference 90 from the terms', scales up to 2^123) 2^8 (a rise it does not follow) 4 (the largest code to a
    token's largest) 2^13 tokens: 2^-67 of the largest.  The bound has 2^-8 of that in the column that holds it."""
    return bound * (1 + 2.0 ** -3) + bound.nan_to_num(0.0).amax(-1, keepdim=True) * 2.0 ** -59


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("dim,shape", PATHS)
@pytest.mark.parametrize("apart", APART)
def test_scales_from_one_end_of_the_range_to_the_other(cuda, dtype, kind, dim, shape, apart):
    """A block of small values counts in the softmax' sum whatever the values beside it weigh."""
    b = _batch(cuda, shape, dim, dtype, kind, seed=len(apart), spread=(-5, -4))
    g = torch.Generator().manual_seed(dim)
    for page, at in _order(b):
        e, louder = APART[apart](torch.arange(len(page)), len(page), g)
        b.cache.v_scale[page, :, at] = torch.exp2(e.float()).to(cuda)[:, None].expand(-1, b.cache.kv_heads)
        b.cache.k_scale[page, :, at] *= louder.to(cuda)[:, None]
    want, bound = b.want()
    close(b.run(out_dtype=F32), want, _wider(bound), f"{shape}, {apart}")


@pytest.mark.parametrize("dtype,kind", KINDS)
def test_a_prefix_and_own_tokens_at_either_end(cuda, dtype, kind):
    """Parts of a row whose references are far apart: what hardly counts in the values does in the sum."""
    for less, more in ((-60, 112), (112, -60), (-60, -1000), (-1000, 112)):
        for shape in ("prefix", "rows_60", "pieces"):
            b = _batch(cuda, shape, 128, dtype, kind, seed=more + 1100, spread=(-5, -4))
            for i, (page, at) in enumerate(_order(b)):
                b.cache.v_scale[page, :, at] = 2.0 ** (more if i else less)
            want, bound = b.want()
            close(b.run(out_dtype=F32), want, _wider(bound), f"{shape}, 2^{less} before 2^{more}")


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("dim,shape", [(64, "prefix"), (128, "chunk_long"), (256, "shared"), (256, "rows_60")])
def test_a_softmax_scale_of_zero(cuda, dtype, kind, dim, shape):
    """Every token that a row sees weighs the same, whatever the queries and the keys' scales."""
    b = _batch(cuda, shape, dim, dtype, kind, seed=dim, spread=(-9, -1), q_spread=3.0)
    want, bound = b.want(scale=0.0)
    other, _ = b.want()
    assert (want - other).abs().max() > 100 * bound.max()  # (another scale would be noticed)
    close(b.run(scale=0.0, out_dtype=F32), want, bound, shape)


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("dim,shape", [(64, "many"), (128, "pieces"), (256, "shared"), (256, "rows_60")])
@pytest.mark.parametrize("share", [1.0, 0.5])
def test_values_up_to_fp32s_largest(cuda, dtype, kind, dim, shape, share):
    """Values of up to 2^127, all or beside the smallest: nothing in between leaves fp32."""
    b = _batch(cuda, shape, dim, dtype, kind, seed=dim, spread=(-5, -4))
    g = torch.Generator().manual_seed(dim)
    for page, at in _order(b):
        e = torch.where(torch.rand(len(page), generator=g) < share, 120.0 if kind == I8 else 118.0, -60.0)
        b.cache.v_scale[page, :, at] = torch.exp2(e).to(cuda)[:, None].expand(-1, b.cache.kv_heads)
    want, bound = b.want()
    got = b.run(out_dtype=F32)
    assert got.isfinite().all()
    close(got, want, _wider(bound), shape)

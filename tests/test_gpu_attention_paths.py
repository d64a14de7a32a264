"""Shared-prefix attention at the borders of its row tiles, lines and paths:
each number of rows that changes how a unit is divided, more sequences than the
lanes or LDS hold, scales of either sign, and what masks, missing pages and
infinities do in each of the paths."""
from __future__ import annotations

import math

import pytest
import torch

from tests import attention_reference as ref
from tests.test_gpu_attention import BF16, E4M3, F16, Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200])
@pytest.mark.parametrize("dim,dtype,cache", [(64, F16, E4M3), (128, BF16, BF16), (256, F16, F16)])
def test_rows_at_the_tiles_borders(cuda, rows, dim, dtype, cache):
    """One head: a new token is a row, of the prefix' units and of the sequence's own."""
    b = Batch(cuda, [rows, 1], [rows + 5, 40], 70, 1, 1, dim, 32, dtype, cache, seed=rows)
    want, bound = b.want()
    ref.close(b.run(), want, bound, f"{rows} rows")
    want, bound = b.want(window=30, sink=3)
    ref.close(b.run(window=30, sink=3), want, bound, f"{rows} rows in a window")


@pytest.mark.parametrize("seqs", [64, 65, 257, 300])
@pytest.mark.parametrize("window", [0, 40])
def test_many_sequences(cuda, seqs, window):
    """More sequences than lanes, and than LDS keeps; some without a new token, some without any."""
    new = [0 if s % 11 == 5 else 1 + (s % 29 == 3) for s in range(seqs)]
    lens = [0 if s % 17 == 6 else max(n, s % 70) for s, n in enumerate(new)]
    b = Batch(cuda, new, lens, 70, 2, 1, 64, 32, F16, F16, seed=seqs)
    want, bound = b.want(window=window, sink=4 if window else 0)
    ref.close(b.run(window=window, sink=4 if window else 0), want, bound, f"{seqs} sequences")


@pytest.mark.parametrize("new", [[1, 2], [20, 3], [90]])
def test_scales_of_either_sign(cuda, new):
    b = Batch(cuda, new, [n + 40 for n in new], 33, 2, 2, 128, 32, F16, F16, seed=13)
    want, bound = b.want(scale=-0.11)
    ref.close(b.run(scale=-0.11), want, bound, "negative")
    # zero: every token that is seen weighs the same (1e-300: zero to the reference too, which takes 0 as unset)
    want, bound = b.want(scale=1e-300)
    ref.close(b.run(scale=0.0), want, bound, "zero")


@pytest.mark.parametrize("max_new", [0, 1, 9, 17, 40])
def test_a_wrong_max_new_only_divides_otherwise(cuda, max_new):
    b = Batch(cuda, [40, 1, 3], [60, 33, 3], 50, 4, 2, 64, 32, F16, F16, seed=14)
    want, bound = b.want()
    ref.close(b.run(max_new=max_new), want, bound, f"max_new {max_new}")


@pytest.mark.parametrize("new", [3, 12, 30, 40])  # 6, 24, 60 and 80 rows: 16-row and shared tiles
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_infinities_that_some_rows_see(cuda, new, bad, dtype):
    """In the values of the middle new token, both signs of an infinity in one column: rows before have neither."""
    b = Batch(cuda, [new], [70], 0, 4, 2, 64, 32, dtype, dtype, seed=15)
    mid = new // 2
    slot = b.cache.slots(b.pages[0], torch.tensor([70 - new + mid, 70 - new + mid + 1], device=cuda))
    k, v = ref.unpack(b.cache, slot)
    clean, bound = b.want()
    v[0, :, 3] = bad
    v[0, :, 40] = bad
    v[1, :, 40] = -bad
    ref.pack(b.cache, slot, k, v)
    got = b.run()
    ref.close(got[:mid], clean[:mid], bound[:mid], "rows before")
    hit = got[mid:, :, 3].double().cpu()
    assert torch.isnan(hit).all() if math.isnan(bad) else (hit == bad).all()
    if mid + 1 < new:
        assert got[mid + 1:, :, 40].isnan().all()  # (+inf and -inf)
    keep = [c for c in range(64) if c not in (3, 40)]
    ref.close(got[mid:][..., keep], clean[mid:][..., keep], bound[mid:][..., keep], "other columns")


@pytest.mark.parametrize("new", [1, 10, 50])  # rows of the prefix: 2, 20 and 100
def test_infinities_of_the_prefix(cuda, new):
    """A NaN of the prefix outside every window reaches nothing; rows that see it have it."""
    b = Batch(cuda, [new], [new], 64, 4, 2, 64, 32, F16, F16, seed=16)
    slot = b.cache.slots(b.prefix_pages, torch.tensor([20], device=cuda))
    k, v = ref.unpack(b.cache, slot)
    clean, bound = b.want(window=44)
    v[0, :, 5] = math.nan
    ref.pack(b.cache, slot, k, v)
    got = b.run(window=44)
    # token j stands at 64 + j and sees positions above 20 + j
    ref.close(got, clean, bound, "outside the window")
    assert b.run()[..., 5].isnan().all()


@pytest.mark.parametrize("new", [1, 12, 45])
@pytest.mark.parametrize("prefix", [0, 64])
def test_pages_outside_the_cache(cuda, new, prefix):
    """Tokens of a page number outside the cache are not there, in own pages and in the prefix."""
    b = Batch(cuda, [new], [100], prefix, 2, 1, 64, 32, F16, F16, seed=17)
    k, v = b.tokens(0)
    where = torch.arange(prefix + 100)
    pos = prefix + 100 - new + torch.arange(new)[:, None]
    gone = (where >= prefix + 32) & (where < prefix + 64)
    pages, prefix_pages = b.pages.clone(), b.prefix_pages.clone()
    b.pages[0, 1] = 10 ** 6
    if prefix:
        b.prefix_pages[0] = -7
        gone |= where < 32
    want, bound = ref.attend(b.q, k, v, (where <= pos) & ~gone, 64 ** -0.5, F16)
    ref.close(b.run(), want, bound, "pages outside the cache")
    b.pages, b.prefix_pages = pages, prefix_pages
    want, bound = b.want()
    ref.close(b.run(), want, bound, "and inside")


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_queries_that_are_not_aligned(cuda, dim):
    """Element-wise query loads in the 16-row, 32-row and shared tiles."""
    for new in ([1, 1], [20, 2], [70]):
        b = Batch(cuda, new, [n + 9 for n in new], 40, 2, 1, dim, 32, BF16, BF16, seed=18)
        want, bound = b.want()
        n = b.q.shape[0]
        odd = torch.empty(n * 2 * (dim + 3) + 1, dtype=BF16, device=cuda)[1:].view(n, 2, dim + 3)[..., :dim]
        b.q = odd.copy_(b.q)
        ref.close(b.run(), want, bound, f"{new}")


@pytest.mark.parametrize("new", [17, 32, 33, 64])
@pytest.mark.parametrize("dim,dtype,cache", [(64, F16, F16), (128, BF16, E4M3), (256, F16, F16)])
def test_rows_of_many_sequences(cuda, new, dim, dtype, cache):
    """17 to 64 rows where there are many units: each wave has 32 of them and its own tiles."""
    b = Batch(cuda, [1] * 70 + [new], [1 + s % 40 for s in range(70)] + [new + 90], 70, 1, 1, dim, 32, dtype, cache,
              seed=new)
    want, bound = b.want()
    ref.close(b.run(), want, bound, f"{new} rows")
    want, bound = b.want(window=30, sink=3)
    ref.close(b.run(window=30, sink=3), want, bound, f"{new} rows in a window")


@pytest.mark.parametrize("new", [24, 60])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_infinities_of_many_sequences(cuda, new, bad, dtype):
    b = Batch(cuda, [new] + [1] * 70, [70] + [5] * 70, 0, 1, 1, 64, 32, dtype, dtype, seed=16)
    mid = new // 2
    slot = b.cache.slots(b.pages[0], torch.tensor([70 - new + mid], device=cuda))
    k, v = ref.unpack(b.cache, slot)
    clean, bound = b.want()
    v[0, :, 3] = bad
    ref.pack(b.cache, slot, k, v)
    got = b.run()
    ref.close(got[:mid], clean[:mid], bound[:mid], "rows before")
    ref.close(got[new:], clean[new:], bound[new:], "other sequences")
    hit = got[mid:new, :, 3].double().cpu()
    assert torch.isnan(hit).all() if math.isnan(bad) else (hit == bad).all()
    keep = [c for c in range(64) if c != 3]
    ref.close(got[mid:new][..., keep], clean[mid:new][..., keep], bound[mid:new][..., keep], "other columns")


@pytest.mark.parametrize("seqs", [1, 8, 9, 32, 33])
@pytest.mark.parametrize("new", [17, 40])
def test_few_and_many_units_of_some_rows(cuda, seqs, new):
    """Two kv heads: up to 32 sequences share tiles, more do not; the workspace of a larger batch serves both."""
    from qwowl35_amd import attention as at

    b = Batch(cuda, [new] + [3] * (seqs - 1), [new + 300] + [3 + 7 * s for s in range(seqs - 1)], 40, 2, 2, 64, 32,
              F16, F16, seed=seqs)
    want, bound = b.want()
    ws = at.prefix_attention_workspace(b.cache, 2, 40, 200)
    ref.close(b.run(workspace=ws), want, bound, f"{seqs} sequences")

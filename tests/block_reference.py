"""A block-scaled cache in float64 on the CPU: its codes and scales from the
documented layout, what an append makes of them, and a batch for attention."""
from __future__ import annotations

import torch

from tests import attention_reference as ref
from tests.test_gpu_attention import Batch, _gen

BLOCK = 32
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
LEAST = 2.0 ** -60


def decode(cache):
    """[(codes [pages, heads, blocks, 32, dim], scales [pages, heads, blocks])] of keys and values, float64."""
    pages, heads, blocks, dim = cache.n_pages, cache.kv_heads, cache.page_size // BLOCK, cache.head_dim
    k = cache.k.cpu().float().double().permute(0, 1, 2, 4, 3, 5).reshape(pages, heads, blocks, BLOCK, dim)
    v = cache.v.cpu().float().double().view(pages, heads, blocks, 4, dim, 8).permute(0, 1, 2, 3, 5, 4)
    return [(k.clone(), cache.k_scale.cpu().double()),
            (v.reshape(pages, heads, blocks, BLOCK, dim).clone(), cache.v_scale.cpu().double())]


def rounded(x, kind):
    """The nearest codes, ties to even; past the largest the largest."""
    x = x.clamp(-TOP[kind], TOP[kind])  # (NaN stays)
    if kind == torch.int8:
        return torch.round(x.nan_to_num(0.0))
    return x.float().to(kind).float().double()


def fitting(m, kind):
    """The least power of two s >= 2^-60 with m <= TOP s; 0 of 0."""
    s = torch.full_like(m, LEAST)
    for _ in range(200):
        s = torch.where(m > TOP[kind] * s, s * 2, s)
    return torch.where(m > 0, s, 0.0)


def append(state, x, slots, kind):
    """One call: tokens x [n, heads, dim] (float64) into ``state`` = (codes, scales), in place."""
    codes, scales = state
    pages, heads, blocks = scales.shape
    by_block: dict = {}
    for t, slot in enumerate(int(s) for s in slots):
        if 0 <= slot < pages * blocks * BLOCK:
            by_block.setdefault(slot // BLOCK, {})[slot % BLOCK] = t
    for block, rows in by_block.items():
        page, at = divmod(block, blocks)
        new = x[list(rows.values())].transpose(0, 1)  # [heads, rows, dim]
        before = scales[page, :, at].clone()
        anew = (before == 0) | (0 in rows)
        m = torch.where(new.isfinite(), new.abs(), 0.0).amax((1, 2))
        now = torch.where(anew, fitting(m, kind), before)
        for _ in range(300):
            now = torch.where(~anew & (m > TOP[kind] * now), now * 2, now)
        shrink = torch.where(anew, 0.0, before / torch.where(now > 0, now, 1.0))
        held = rounded(codes[page, :, at] * torch.where(anew, 1.0, shrink)[:, None, None], kind)
        held[anew] = 0.0
        new = new.clamp(-3.4e38, 3.4e38)
        over = torch.where((now > 0)[:, None, None], new / torch.where(now > 0, now, 1.0)[:, None, None], new * 0.0)
        held[:, list(rows)] = rounded(over, kind)
        codes[page, :, at], scales[page, :, at] = held, now


def fill(cache, randn, scaled=0.6, spread=(-7, -2)):
    """Random codes everywhere; scales of a share of the blocks, powers of two, zero elsewhere."""
    kind, device = cache.k.dtype, cache.k.device
    for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x = randn(*codes.shape) * TOP[kind] * 0.25
        x = x.clamp(-TOP[kind], TOP[kind])
        codes.copy_(x.round().to(kind) if kind == torch.int8 else x.to(kind))
        e = torch.randint(*spread, scale.shape, device=device)
        scale.copy_(torch.exp2(e.float()) * (torch.rand(scale.shape, device=device) < scaled))


def same(cache, want, what=""):
    for name, (codes, scales), (wc, ws) in zip(("keys", "values"), decode(cache), want):
        assert torch.equal(scales, ws), f"{what}: scales of {name}: {(scales != ws).sum()} differ"
        off = ~((codes == wc) | (codes.isnan() & wc.isnan()))
        assert not off.any(), f"{what}: {int(off.sum())} codes of {name} differ, first at {off.nonzero()[0].tolist()}"


def close(got, want, bound, what=""):
    """As over other caches, and NaN where the formula has NaN (an e4m3 code past 448 is one)."""
    nan = want.isnan()
    assert torch.equal(got.isnan().cpu(), nan), f"{what}: NaN in other places than the formula's"
    ref.close(got.cpu().masked_fill(nan, 0.0), want.masked_fill(nan, 0.0), bound.masked_fill(nan, 0.0), what)


class BlockBatch(Batch):
    """A batch over shuffled pages of a block-scaled cache.  Blocks that hold no token have a scale of NaN; slots
    behind the last token hold NaN (e4m3) or the largest code."""

    def __init__(self, cuda, new, lens, prefix, heads, kv_heads, dim, page, dtype, kind, seed=0, spread=(-7, -3),
                 q_spread=1.0):
        from qwowl35_amd import attention as at

        super().__init__(cuda, new, [0] * len(lens), 0, heads, kv_heads, dim, page, dtype, dtype, seed)
        self.lens, self.prefix = lens, prefix
        count = lambda n: (n + page - 1) // page  # noqa: E731
        per = max([count(n) for n in lens] + [1])
        total = count(prefix) + sum(count(n) for n in lens) + 2
        self.cache = c = at.PagedCache.empty(total, kv_heads, page, dim, kind, device=cuda, block_scales=True)
        randn = _gen(cuda, seed + 1)
        for t in (c.k, c.v):
            t.view(torch.uint8).fill_(0x7f)
        c.k_scale.fill_(float("nan"))
        c.v_scale.fill_(float("nan"))
        order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        self.prefix_pages = order[:count(prefix)].to(cuda)
        table, at_ = torch.full((len(lens), per), -1, dtype=torch.int32), count(prefix)
        for s, n in enumerate(lens):
            table[s, :count(n)] = order[at_:at_ + count(n)]
            at_ += count(n)
        self.pages = table.to(cuda)
        self.lengths = torch.tensor(lens, dtype=torch.int32, device=cuda)
        self.q = (self.q.float() * q_spread).to(dtype)
        g = torch.Generator(device=cuda).manual_seed(seed + 2)
        for pages, n in [(self.prefix_pages, prefix)] + [(self.pages[s], n) for s, n in enumerate(lens)]:
            if not n:
                continue
            slots = c.slots(pages, torch.arange(n, device=cuda))
            size = TOP[kind] * 0.25
            ref.pack(c, slots, (randn(n, kv_heads, dim) * size).round(), (randn(n, kv_heads, dim) * size).round())
            b = torch.unique(slots // BLOCK)
            for scale in (c.k_scale, c.v_scale):
                e = torch.randint(*spread, (b.numel(), kv_heads), generator=g, device=cuda)
                if kind != torch.int8:
                    e -= 2
                scale[b // (page // BLOCK), :, b % (page // BLOCK)] = torch.exp2(e.float())

    def tokens(self, s):
        parts = []
        for pages, n in [(self.prefix_pages, self.prefix), (self.pages[s], self.lens[s])]:
            slots = self.cache.slots(pages, torch.arange(n, device=pages.device)).cpu()
            page, at = slots // self.cache.page_size, slots % self.cache.page_size
            both = []
            for codes, scales in self.decoded():
                both.append(codes[page, :, at // BLOCK, at % BLOCK] * scales[page, :, at // BLOCK][..., None])
            parts.append(both)
        return [torch.cat([p[i] for p in parts]) for i in range(2)]

    def decoded(self):
        if getattr(self, "_decoded", None) is None:
            self._decoded = decode(self.cache)
        return self._decoded

    def want(self, window=0, sink=0, scale=None, gate=None):
        """(out, bound) from the formula, row by row."""
        heads, dim = self.q.shape[1:]
        scale = dim ** -0.5 if scale is None else scale
        group = heads // self.cache.kv_heads
        out = torch.zeros(self.q.shape, dtype=torch.float64)
        bound = torch.zeros_like(out)
        q = self.q.double().cpu()
        first = 0
        for s, (new, length) in enumerate(zip(self.new, self.lens)):
            k, v = self.tokens(s)
            where = torch.arange(self.prefix + length)
            for j in range(new):
                pos = self.prefix + length - new + j
                seen = where <= pos
                if window:
                    seen &= (where > pos - window) | (where < sink)
                if not seen.any():
                    continue
                ks, vs = k[seen], v[seen]
                for h in range(heads):
                    kh, vh = ks[:, h // group], vs[:, h // group]
                    row = q[first + j, h]
                    p = torch.softmax((kh @ row) * scale, 0)
                    off = float((kh.abs() @ row.abs()).max()) * abs(scale) * (dim + 4) * 2.0 ** -24
                    out[first + j, h] = p @ vh
                    # Weights: rounded to the queries' type, exponentials and rescalings to 2^-18, twice the logits'
                    # error; log2 of a scale of up to 2^+-60 within two steps, its sum with the reference and the
                    # exponent's, each of less than 2^7: together under 2^-16.  A weight counts what its values
                    # weigh; those under fp16's least (2^-25, the reference 2^7 below the row's largest) are lost,
                    # and the largest code stands for at most four times a token's largest value.
                    lost = 2.0 ** -32 if self.dtype == torch.float16 else 0.0
                    bound[first + j, h] = ((ref.EPS[self.dtype] + 2.0 ** -18 + 2.0 ** -16 + 2 * off) * (p @ vh.abs())
                                           + lost * p.numel() * 4 * float((p * vh.nan_to_num(0.0).abs().amax(1)).max()))
            first += new
        if gate is not None:
            g = torch.sigmoid(gate.double().cpu())
            out, bound = out * g, bound * g + (out * g).abs() * 2.0 ** -20  # (exp, sum and quotient of the gate)
        return out, bound

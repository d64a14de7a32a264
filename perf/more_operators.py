"""The 8-bit cache with a scale for each block of tokens and head, as cases that can be timed and compared.

Keys and values of a paged cache are int8 or e4m3 codes; a block of 32 tokens
(slot // 32) of a kv head has a scale of its own, for its keys and for its
values, and a code stands for itself times it.  ``kv_append`` quantises tokens as
it writes them, ``kv_read`` reads them back, ``prefix_attention`` attends over
them.  ``own`` false computes the three in plain torch, true calls the library.

Appending: with m the largest magnitude of the block's new tokens and Q the
largest code (127, 448), the block's scale becomes the least power of two s with
m <= Q s, or stays if it is larger; tokens that the block held before are rounded
to the new scale.  Writing a block's first token begins it anew: what it held is
zero.  (A scale is at least 2^-60, and zero where a block holds zeros only.)

The pages' layout is the library's: for each kv head keys as
[page / 32][D / 8][32 tokens][8 columns] and values as [page / 8][D][8 tokens];
scales are fp32 [pages][kv heads][page / 32].  Token j of a sequence whose page
list is p lies in slot p[j // page] * page + j % page.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BLOCK = 32
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn,
          "i8": torch.int8}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1, "i8": 1}
TOP = {"e4m3": 448.0, "i8": 127.0}  # the largest code
LEAST = -60                        # the least scale's exponent
EPS = 1e-6


# ---- the cases ---------------------------------------------------------------------------------------------------

def listed() -> list[dict]:
    return [
        # one decode step of eight sequences, each somewhere in its block, and what their blocks then hold
        _append("append_b8_i8", 8, 1, 13, 4, 256, 64, [11, 11, 10], True, "f32", "i8", page=64, norm=True),
        # a prefill chunk's odd remainder that continues a block
        _append("append_chunk_e4m3", 1, 249, 77, 4, 256, 64, [11, 11, 10], True, "f32", "e4m3", page=128, norm=True),
        # a long prompt, bf16 in, another head layout
        _append("append_long_i8", 1, 8192, 0, 8, 128, 128, [16, 24, 24], False, "bf16", "i8", page=256, norm=False),
        # the last tokens of a sequence, to be looked at or written elsewhere
        _read("read_tail_i8", 45, 4, 256, "i8", "f16", page=64),
        # a whole document's cache on its way to a 16-bit one
        _read("read_long_e4m3", 20011, 8, 128, "e4m3", "bf16", page=256),
        # one sequence, early in its answer, no shared prefix: latency
        _attend("decode_b1_short_i8", 1, [1], 0, [517], 16, 4, 256, "f16", "i8", page=64, gate="f32"),
        # eight sequences after one system prompt
        _attend("decode_b8_prefix_i8", 8, [1], 8191, [37, 600, 1, 255, 130, 512, 33, 64], 16, 4, 256, "f16", "i8",
                page=64, gate="f32"),
        # five answers about one long document
        _attend("decode_b5_long_i8", 5, [1], 100003, [1, 2900, 800, 127, 1500], 16, 4, 256, "f16", "i8", page=256,
                gate="f32"),
        # a full serving batch after a shared prompt, another head layout, bf16 queries
        _attend("decode_b64_e4m3", 64, [1], 16384, [1 + (37 * s * s) % 500 for s in range(64)], 32, 8, 128, "bf16",
                "e4m3", page=128, gate=""),
        # the next chunk of a prompt that continues a shared prefix
        _attend("chunk_256_prefix_i8", 1, [256], 16001, [700], 16, 4, 256, "f16", "i8", page=256, gate="f32"),
        # drafted tokens checked under a sliding window with attention sinks
        _attend("verify_b4_window_e4m3", 4, [5, 1, 9, 4], 0, [30001, 5000, 12345, 20], 16, 4, 256, "bf16", "e4m3",
                page=4096, gate="", window=4096, sink=64),
        # short narrow-headed sequences, a few drafted tokens each
        _attend("verify_b24_d64_i8", 24, [3], 0, [5 + (131 * s) % 2000 for s in range(24)], 14, 2, 64, "f16", "i8",
                page=96, gate="f16"),
    ]


def _text(numbers) -> str:
    """A case's list, as text: ``_lists`` reads it back."""
    return " ".join(str(v) for v in numbers)


def _lists(case: dict) -> dict:
    return case | {key: [int(v) for v in case[key].split()] for key in ("sections", "new", "lens")
                   if isinstance(case.get(key), str)}


def _append(name, seqs, each, first, heads, dim, rot, sections, interleaved, dtype, cache, page, norm):
    """``each`` new tokens for every sequence; sequence i has 37 i + ``first`` tokens in its first page already."""
    return {"name": name, "kind": "append", "seqs": seqs, "each": each, "first": first, "heads": heads, "dim": dim,
            "rot": rot, "sections": _text(sections), "interleaved": interleaved, "dtype": dtype, "cache": cache,
            "page": page, "norm": norm}


def _read(name, n, heads, dim, cache, out, page):
    return {"name": name, "kind": "read", "n": n, "heads": heads, "dim": dim, "cache": cache, "out": out, "page": page}


def _attend(name, seqs, new, prefix, lens, heads, kv_heads, dim, dtype, cache, page, gate, window=0, sink=0):
    """Per sequence ``new`` new tokens, ``lens`` own ones (the new ones among them), after ``prefix`` shared ones."""
    new = new * seqs if len(new) == 1 else new
    return {"name": name, "kind": "attend", "new": _text(new), "prefix": prefix, "lens": _text(lens),
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "cache": cache, "page": page,
            "gate": gate, "window": window, "sink": sink}


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["append", "append", "read", "attend", "attend", "attend"])
    dim, cache, page = rng.choice([64, 128, 256]), rng.choice(["i8", "e4m3"]), rng.choice([32, 64, 96, 256, 4096])
    flip = lambda: rng.random() < 0.5  # noqa: E731
    if kind == "append":
        heads, rot = rng.choice([1, 2, 3, 4, 8]), rng.choice([dim, dim // 2, dim // 4])
        third = rot // 2 // 3
        sections = rng.choice([[], [rot // 2 - 2 * third, third, third]])
        seqs = _log_int(rng, 1, 64)
        each = _log_int(rng, 1, 8192 // seqs) if flip() else rng.randint(1, 8)
        c = _append("", seqs, each, rng.randrange(page), heads, dim, rot, sections, flip(),
                    rng.choice(["f32", "f16", "bf16"]), cache, page, flip())
    elif kind == "read":
        c = _read("", _log_int(rng, 1, 20011), rng.choice([1, 2, 3, 4, 8]), dim, cache,
                  rng.choice(["f16", "bf16"]), page)
    else:
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 6, 8])
        seqs = _log_int(rng, 1, 64)
        most = _log_int(rng, 1, max(1, 256 // seqs)) if flip() else 1
        new = [rng.randint(1, most) for _ in range(seqs)]
        prefix = _log_int(rng, 1, 100000) if rng.random() < 0.7 else 0
        top = _log_int(rng, most, 4096 if prefix else 32768)
        lens = [max(k, _log_int(rng, 1, top)) for k in new]
        dtype = "f16" if cache == "i8" else rng.choice(["f16", "bf16"])
        window, sink = (_log_int(rng, 16, 8192), rng.choice([0, 4, 64])) if rng.random() < 0.25 else (0, 0)
        c = _attend("", seqs, new, prefix, lens, heads, kv_heads, dim, dtype, cache, page,
                    rng.choice(["", "f32", dtype]), window, sink)
        flops, size = (max(work(x)[key] for x in listed()) for key in ("flops", "bytes"))
        while (work(c)["flops"] > flops or work(c)["bytes"] > size or seqs * max(lens) * kv_heads * dim > 1 << 28
               or seqs * max(new) * heads * (c["prefix"] + max(lens)) > 1 << 29):  # (what the plain form holds)
            lens = [max(k, v // 2) for k, v in zip(new, lens)]
            c |= {"prefix": c["prefix"] // 2, "lens": _text(lens)}
    del c["name"]
    return c


def _spans(c: dict) -> list[tuple]:
    """Of an append's sequences: (tokens held before, its first block, the end of its blocks)."""
    at = [(37 * i + c["first"]) % c["page"] for i in range(c["seqs"])]
    return [(a, a // BLOCK, -(-(a + c["each"]) // BLOCK)) for a in at]


def work(case: dict) -> dict:
    c = _lists(case)
    if c["kind"] == "append":
        n = c["seqs"] * c["each"]
        row, axes = c["heads"] * c["dim"] * 2, len(c["sections"]) or 1
        held = sum(hi - lo for _, lo, hi in _spans(c)) * BLOCK
        # tokens in and codes out; what the blocks then hold, once
        return {"bytes": n * row * (SIZE[c["dtype"]] + 1) + (8 + 4 * axes) * n + held * row * 2,
                "flops": n * row / 2 * (3 * c["rot"] / c["dim"] + (4 if c["norm"] else 0) + 6)}
    if c["kind"] == "read":
        n = c["n"] * c["heads"] * c["dim"] * 2
        return {"bytes": n * (1 + SIZE[c["out"]]) + 8 * c["n"], "flops": n}
    pairs, seen = 0, 0
    for new, length in zip(c["new"], c["lens"]):
        for j in range(new):
            pos = c["prefix"] + length - new + j
            pairs += pos + 1 - (max(0, pos + 1 - c["window"] - c["sink"]) if c["window"] else 0)
    if c["window"]:  # what any row of the batch sees of the prefix, and of each sequence's own tokens
        span = [(p + n - k, p + n) for p, n, k in ((c["prefix"], n, k) for n, k in zip(c["lens"], c["new"]))]
        for (first, end), length in zip(span, c["lens"]):
            low = max(c["prefix"], first + 1 - c["window"])
            seen += end - low + max(0, min(c["sink"], low) - c["prefix"])
        low = max(0, min(first + 1 - c["window"] for first, _ in span))
        seen += max(0, c["prefix"] - low) + min(c["sink"], low, c["prefix"])
    else:
        seen = c["prefix"] + sum(c["lens"])
    rows = sum(c["new"]) * c["heads"] * c["dim"]
    return {"bytes": seen * c["kv_heads"] * 2 * (c["dim"] + 4 / BLOCK) + rows * 2 * SIZE[c["dtype"]]
            + (rows * SIZE[c["gate"]] if c["gate"] else 0),
            "flops": 4 * c["heads"] * c["dim"] * pairs}


# ---- what a program has in hand before the call ------------------------------------------------------------------

def _generator(seed: int) -> torch.Generator:
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _cache(s: dict, c: dict, g, pages: int, heads: int) -> None:
    """A cache in use: codes of normal values, the scales of a block's spread (a factor of four from block to block)."""
    d, page, kind = c["dim"], c["page"], DTYPES[c["cache"]]
    spread = 30.0 if c["cache"] == "i8" else 110.0

    def codes(*shape):
        x = torch.randn(shape, generator=g, device=DEV).mul_(spread).clamp_(-TOP[c["cache"]], TOP[c["cache"]])
        return x.round_().to(kind) if kind == torch.int8 else x.to(kind)

    def scales():
        e = torch.randint(-6, -3, (pages, heads, page // BLOCK), generator=g, device=DEV)
        return torch.exp2((e - (0 if c["cache"] == "i8" else 2)).float())

    s["cache_k"] = codes(pages, heads, page // BLOCK, d // 8, BLOCK, 8)
    s["cache_v"] = codes(pages, heads, page // 8, d, 8)
    s["k_scale"], s["v_scale"] = scales(), scales()
    if own:  # the handle over these tensors that a program keeps
        from qwowl35_amd import attention as at_

        s["cache"] = at_.PagedCache(s["cache_k"], s["cache_v"], s["k_scale"], s["v_scale"])


def prepare(case: dict, seed: int):
    c, g = _lists(case), _generator(seed)
    s: dict = {"case": c}
    return {"append": _prepare_append, "read": _prepare_read, "attend": _prepare_attend}[c["kind"]](c, s, g)


def _prepare_append(c, s, g):
    normal = lambda *shape: torch.randn(shape, generator=g, device=DEV)  # noqa: E731
    page, h, d = c["page"], c["heads"], c["dim"]
    spans = _spans(c)
    count = [-(-(a + c["each"]) // page) for a, _, _ in spans]
    _cache(s, c, g, sum(count) + 1, h)
    order = torch.randperm(sum(count) + 1, generator=g, device=DEV).cpu()
    slots, touched, used = [], [], 0
    for (a, lo, hi), pages in zip(spans, count):
        mine, used = order[used:used + pages], used + pages
        for at, to in ((torch.arange(a, a + c["each"]), slots), (torch.arange(lo * BLOCK, hi * BLOCK), touched)):
            to.append(mine[at // page] * page + at % page)
    s["slots"], s["touched"] = torch.cat(slots).to(DEV), torch.cat(touched).to(DEV)
    # each sequence far into a context of its own; a long prompt's second quarter is an image in rows and columns
    start = torch.randint(0, 200000, (c["seqs"], 1), generator=g, device=DEV)
    t = start + torch.arange(c["each"], device=DEV)
    if c["sections"]:
        lo, hi = c["each"] // 4, c["each"] // 2
        wide = max(1, math.isqrt(max(1, hi - lo)))
        cell = torch.arange(c["each"], device=DEV) - lo
        image = (cell >= 0) & (cell < hi - lo)
        t = torch.stack([torch.where(image, start + lo, t), torch.where(image, start + lo + cell // wide, t),
                         torch.where(image, start + lo + cell % wide, t)]).flatten(1)
    else:
        t = t.flatten()
    s["positions"] = t.to(torch.int32).contiguous()
    s["norm"] = torch.rand(d, generator=g, device=DEV) + 0.5 if c["norm"] else None
    n = c["seqs"] * c["each"]
    s["k"], s["v"] = normal(n, h, d).to(DTYPES[c["dtype"]]), normal(n, h, d).to(DTYPES[c["dtype"]])
    if own:
        from qwowl35_amd import attention as at_

        s["rope"] = at_.Rotary(c["rot"], 1e7, c["sections"], c["interleaved"], device=DEV)
    return s


def _prepare_read(c, s, g):
    """The last ``n`` tokens of a sequence that ends in the middle of a page."""
    page = c["page"]
    pages = -(-(c["n"] + page // 3) // page) + 1
    _cache(s, c, g, pages + 1, c["heads"])
    order = torch.randperm(pages + 1, generator=g, device=DEV)
    end = pages * page - page // 2
    at = torch.arange(end - c["n"], end, device=DEV)
    s["slots"] = order[at // page] * page + at % page
    return s


def _prepare_attend(c, s, g):
    d, page = c["dim"], c["page"]
    count = lambda n: (n + page - 1) // page  # noqa: E731
    seqs, total = len(c["new"]), sum(c["new"])
    own_pages = [count(n) for n in c["lens"]]
    pages = count(c["prefix"]) + sum(own_pages) + 1
    normal = lambda *shape: torch.randn(shape, generator=g, device=DEV)  # noqa: E731
    _cache(s, c, g, pages, c["kv_heads"])
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    s["prefix_pages"] = order[:count(c["prefix"])].contiguous()
    table = torch.zeros((seqs, max(own_pages)), dtype=torch.int32)
    at, order = count(c["prefix"]), order.cpu()
    for i, k in enumerate(own_pages):
        table[i, :k] = order[at:at + k]
        at += k
    s["pages"] = table.to(DEV)
    s["lengths"] = torch.tensor(c["lens"], dtype=torch.int32, device=DEV)
    starts = [0]
    for k in c["new"]:
        starts.append(starts[-1] + k)
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
    # queries that single some keys out: logits of standard deviation 1 to 4
    s["q"] = (normal(total, c["heads"], d) * 2).to(DTYPES[c["dtype"]])
    s["gate"] = None
    if c["gate"]:  # the gate half of each head of the q projection
        s["gate"] = normal(total, c["heads"], 2 * d).to(DTYPES[c["gate"]])[..., d:]
    if own:
        from qwowl35_amd import attention as at_

        s["workspace"] = at_.prefix_attention_workspace(s["cache"], c["heads"], seqs, total, device=DEV)
        s["max_new"] = max(c["new"])
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------

def run(s):
    c = s["case"]
    if own:
        from qwowl35_amd import attention as at_

        if c["kind"] == "append":
            at_.kv_append(s["cache"], s["k"], s["v"], s["slots"], rope=s["rope"], positions=s["positions"],
                          norm=s["norm"], eps=EPS)
            return at_.kv_read(s["cache"], s["touched"], dtype=torch.float16)
        if c["kind"] == "read":
            return at_.kv_read(s["cache"], s["slots"], dtype=DTYPES[c["out"]])
        return at_.prefix_attention(s["q"], s["cache"], s["pages"], s["lengths"], s["starts"],
                                    max_new=s["max_new"], prefix_pages=s["prefix_pages"], prefix_len=c["prefix"],
                                    window=c["window"], sink=c["sink"], gate=s["gate"], workspace=s["workspace"])
    return {"append": _plain_append, "read": _plain_read, "attend": _plain_attend}[c["kind"]](c, s)


def _plain_rotate(c, x, positions, norm):
    """RMS norm and rotation in float32; the angles, positions times frequencies, in float64."""
    x = x.float()
    if norm is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * norm
    half, r = c["rot"] // 2, c["rot"]
    pair = torch.arange(half, device=DEV)
    freq = torch.pow(1e7, pair.double() * (-2.0 / r))
    if c["sections"]:
        _, sh, sw = c["sections"]
        if c["interleaved"]:  # pairs take the axes in turn, as far as each axis' section reaches
            axis = pair % 3
            axis = torch.where(((axis == 1) & (pair < 3 * sh)) | ((axis == 2) & (pair < 3 * sw)), axis, 0)
        else:
            axis = (pair >= c["sections"][0]).long() + (pair >= c["sections"][0] + sh).long()
        pos = positions[axis].t()
    else:
        pos = positions[:, None]
    angle = pos.double() * freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[..., :half], x[..., half:r]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., r:]], -1)


def _bytes(x):
    """8-bit floats as bytes: indexing takes no other 8-bit type."""
    return x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x


def _keys(s):
    """Cache keys as [pages, page / 32, 32, heads, D / 8, 8], a view."""
    return _bytes(s["cache_k"]).permute(0, 2, 4, 1, 3, 5)


def _values(s):
    """Cache values as [pages, page / 32, 4, 8, heads, D], a view."""
    v = _bytes(s["cache_v"])
    return v.view(v.shape[0], v.shape[1], -1, 4, *v.shape[3:]).permute(0, 2, 3, 5, 1, 4)


def _plain_append(c, s):
    """Block by block: old tokens as they stand with the new ones in their places, over the scale that both fit."""
    kind, h, d, top = DTYPES[c["cache"]], c["heads"], c["dim"], TOP[c["cache"]]
    block = s["touched"].view(-1, BLOCK)[:, 0] // BLOCK  # the blocks that are written to
    page, at = block // (c["page"] // BLOCK), block % (c["page"] // BLOCK)
    order = torch.argsort(block)
    place = order[torch.searchsorted(block[order], s["slots"] // BLOCK)]  # of each token: its block, and its row there
    row = s["slots"] % BLOCK
    count = block.shape[0]
    new = torch.zeros((count, BLOCK), dtype=torch.bool, device=DEV)
    new[place, row] = True
    anew = new[:, :1]
    out = []
    for x, view, scale in ((_plain_rotate(c, s["k"], s["positions"], s["norm"]), _keys(s), s["k_scale"]),
                           (s["v"].float(), _values(s), s["v_scale"])):
        was = scale[page, :, at] * ~anew                            # [blocks, heads]
        codes = view[page, at]
        old = codes.reshape(count, BLOCK, h, d).view(kind).float() * was[:, None, :, None]
        both = old.masked_fill(anew[:, :, None, None], 0)
        both[place, row] = x
        m = (both * new[:, :, None, None]).abs().amax((1, 3))
        mantissa, exponent = torch.frexp(m)                         # m = mantissa 2^exponent, mantissa from 1/2 up
        need = exponent - math.frexp(top)[1] + (mantissa > math.frexp(top)[0]).int()
        need = torch.exp2(need.clamp_min(LEAST).float()) * (m > 0)
        now = torch.maximum(was, need)
        over = (both / torch.where(now > 0, now, 1.0)[:, None, :, None]).clamp(-top, top)
        over = over.round().to(kind) if kind == torch.int8 else over.to(kind)
        view[page, at] = _bytes(over).view(codes.shape)
        scale[page, :, at] = now
        out.append((over.float() * now[:, None, :, None]).to(torch.float16).view(-1, h, d))
    return tuple(out)


def _plain_read(c, s):
    kind, n, out = DTYPES[c["cache"]], c["n"], DTYPES[c["out"]]
    page, at = s["slots"] // c["page"], s["slots"] % c["page"]
    k = _keys(s)[page, at // BLOCK, at % BLOCK].reshape(n, c["heads"], -1).view(kind).float()
    v = _values(s)[page, at // BLOCK, at % BLOCK // 8, at % 8].view(kind).float()
    return ((k * s["k_scale"][page, :, at // BLOCK][..., None]).to(out),
            (v * s["v_scale"][page, :, at // BLOCK][..., None]).to(out))


def _tokens(c, s, pages):
    """Keys and values [..., tokens, heads, D] in float32 of pages [..., m]."""
    kind, lead = DTYPES[c["cache"]], pages.shape[:-1]
    pages = pages.long()
    shape = (*lead, pages.shape[-1] * c["page"], c["kv_heads"], c["dim"])
    sk, sv = (x[pages].transpose(-1, -2) for x in (s["k_scale"], s["v_scale"]))  # [..., m, page / 32, heads]
    k = _keys(s)[pages].view(kind).float() * sk[..., None, :, None, None]
    v = _values(s)[pages].view(kind).float() * sv[..., None, None, :, None]
    return k.reshape(shape), v.reshape(shape)


def _plain_attend(c, s):
    """Ragged queries padded to [sequence, new, ...]; scores over prefix and own tokens side by side, one softmax."""
    heads, hk, d, total = c["heads"], c["kv_heads"], c["dim"], s["q"].shape[0]
    group, p, seqs = heads // hk, c["prefix"], s["lengths"].shape[0]
    new = (s["starts"][1:] - s["starts"][:-1]).long()
    most, longest = max(c["new"]), max(c["lens"])
    token = torch.arange(total, device=DEV)
    seq = torch.searchsorted(s["starts"][1:].long(), token, right=True)
    place = token - s["starts"].long()[seq]
    q = torch.zeros((seqs, most, heads, d), device=DEV)
    q[seq, place] = s["q"].float() / math.sqrt(d)
    pk, pv = _tokens(c, s, s["prefix_pages"])
    ok, ov = _tokens(c, s, s["pages"])
    pk, pv, ok, ov = pk[:p], pv[:p], ok[:, :longest], ov[:, :longest]
    q = q.view(seqs, most, hk, group, d).permute(2, 0, 3, 1, 4)  # [hk, seqs, group, most, d]
    rows = group * most
    sp = torch.matmul(q.reshape(hk, seqs * rows, d), pk.permute(1, 2, 0).contiguous())
    sp = sp.view(hk, seqs, group, most, p)
    so = torch.matmul(q.reshape(hk, seqs, rows, d), ok.permute(2, 0, 3, 1).contiguous())
    scores = torch.cat([sp, so.view(hk, seqs, group, most, longest)], -1)
    where = torch.arange(p + longest, device=DEV)
    pos = p + s["lengths"].long()[:, None] - new[:, None] + torch.arange(most, device=DEV)  # [seqs, most]
    seen = where <= pos[..., None]
    if c["window"]:
        seen = seen & ((where > pos[..., None] - c["window"]) | (where < c["sink"]))
    scores = scores.masked_fill_(~seen[:, None], float("-inf"))
    top = scores.amax(-1, keepdim=True).clamp_min(-3e38)
    e = (scores - top).exp_()
    norm = e.sum(-1, keepdim=True)
    e = e / torch.where(norm > 0, norm, 1.0)
    out = torch.matmul(e[..., :p].reshape(hk, seqs * rows, p), pv.permute(1, 0, 2).contiguous()).view(hk, seqs, rows, d)
    out = out + torch.matmul(e[..., p:].reshape(hk, seqs, rows, longest), ov.permute(2, 0, 1, 3).contiguous())
    out = out.view(hk, seqs, group, most, d).permute(1, 3, 0, 2, 4).reshape(seqs, most, heads, d)[seq, place]
    if s["gate"] is not None:
        out = out * torch.sigmoid(s["gate"].float())
    return out.to(DTYPES[c["dtype"]])


# ---- from the definition, in 64 bits -----------------------------------------------------------------------------

def exact(case: dict, seed: int):
    s = prepare(case, seed)
    c = s["case"]
    return {"append": _exact_append, "read": _exact_read, "attend": _exact_attend}[c["kind"]](c, s)


def _exact_rotate(c, x, positions, norm):
    """The rotated part of a head as complex numbers x_i + i x_(i + rot/2), each turned by its angle."""
    x, half = x.double(), c["rot"] // 2
    if norm is not None:
        x = x / ((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * norm.double()
    angle = torch.empty((x.shape[0], half), dtype=torch.float64, device=DEV)
    left = list(c["sections"][1:]) + [0, 0]
    for i in range(half):
        if not c["sections"]:
            at = positions
        elif c["interleaved"]:
            axis = i % 3 if i % 3 and i // 3 < left[i % 3 - 1] else 0
            at = positions[axis]
        else:
            at = positions[sum(i >= sum(c["sections"][:k]) for k in (1, 2))]
        angle[:, i] = at.double() * (1e7 ** (-2.0 * i / c["rot"]))
    z = torch.complex(x[..., :half], x[..., half:2 * half]) * torch.polar(torch.ones_like(angle), angle)[:, None]
    y = x.clone()
    y[..., :half], y[..., half:2 * half] = z.real, z.imag
    return y


def _decoded(c, s, slots, heads):
    """(keys, values, index of their codes) [heads, tokens, D] of slots, by the layout's arithmetic."""
    d, page, kind = c["dim"], c["page"], DTYPES[c["cache"]]
    col, head = torch.arange(d, device=DEV), torch.arange(heads, device=DEV)[:, None, None]
    pg, t = (slots.long() // page)[:, None], (slots.long() % page)[:, None]
    base = (pg * heads + head) * page * d
    where = (base + (t // 32) * 32 * d + (col // 8) * 256 + (t % 32) * 8 + col % 8,
             base + (t // 8) * 8 * d + col * 8 + t % 8)
    block = ((pg * heads + head) * (page // BLOCK) + t // BLOCK)  # [heads, tokens, 1]
    found = []
    for codes, scale, at in ((s["cache_k"], s["k_scale"], where[0]), (s["cache_v"], s["v_scale"], where[1])):
        raw = codes.view(torch.uint8).view(-1)[at].view(kind).double()
        found.append(raw * scale.double().view(-1)[block])
    return (*found, block[..., 0])


def _to_grid(c, x):
    """The nearest code, ties to even."""
    if c["cache"] == "i8":
        return torch.round(x).clamp(-127, 127)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)  # (subnormals share the least step)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _exact_append(c, s):
    """Head by head, every token of the touched blocks: what the block held, replaced where the call writes."""
    h, d = c["heads"], c["dim"]
    k_old, v_old, block = _decoded(c, s, s["touched"], h)
    count = s["touched"].shape[0] // BLOCK
    slot_of = {int(v): i for i, v in enumerate(s["touched"].tolist())}
    at = torch.tensor([slot_of[int(v)] for v in s["slots"].tolist()], device=DEV)
    written = torch.zeros(count * BLOCK, dtype=torch.bool, device=DEV)
    written[at] = True
    anew = written.view(count, BLOCK)[:, 0].repeat_interleave(BLOCK)
    out = []
    for x, old, scale in ((_exact_rotate(c, s["k"], s["positions"], s["norm"]), k_old, s["k_scale"]),
                          (s["v"].double(), v_old, s["v_scale"])):
        full = torch.zeros((h, count * BLOCK, d), dtype=torch.float64, device=DEV)
        full[:, at] = x.transpose(0, 1)
        m = full.abs().view(h, count, -1).amax(-1)
        need = torch.full_like(m, 2.0 ** LEAST)
        for _ in range(200):  # doubled until the largest fits
            need = torch.where(m > TOP[c["cache"]] * need, need * 2, need)
        need = torch.where(m > 0, need, 0.0)
        was = torch.where(anew.view(count, BLOCK)[:, 0], 0.0, scale.double().view(-1)[block].view(h, count, BLOCK)[..., 0])
        now = torch.maximum(was, need).repeat_interleave(BLOCK, -1)[..., None]
        value = torch.where(written[:, None], full, torch.where(anew[:, None], 0.0, old))
        code = _to_grid(c, value / torch.where(now > 0, now, 1.0))
        out.append((code * now).transpose(0, 1))
    return tuple(out)


def _exact_read(c, s):
    k, v, _ = _decoded(c, s, s["slots"], c["heads"])
    return k.transpose(0, 1), v.transpose(0, 1)


def _exact_attend(c, s):
    """Sequence by sequence: its tokens' keys and values as one list, each new token's softmax over what it sees."""
    group, d, page = c["heads"] // c["kv_heads"], c["dim"], c["page"]

    def slots(pages, n):
        t = torch.arange(n, device=DEV)
        return pages.long()[t // page] * page + t % page if n else t

    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    prefix = _decoded(c, s, slots(s["prefix_pages"], c["prefix"]), c["kv_heads"])
    first = 0
    for i, (new, length) in enumerate(zip(c["new"], c["lens"])):
        mine = _decoded(c, s, slots(s["pages"][i], length), c["kv_heads"])
        at = torch.arange(c["prefix"] + length, device=DEV)
        pos = c["prefix"] + length - new + torch.arange(new, device=DEV)[:, None]
        seen = at <= pos
        if c["window"]:
            seen &= (at > pos - c["window"]) | (at < c["sink"])
        for h in range(c["kv_heads"]):
            k = torch.cat([prefix[0][h], mine[0][h]])
            v = torch.cat([prefix[1][h], mine[1][h]])
            for j in range(h * group, (h + 1) * group):
                score = (s["q"][first:first + new, j].double() @ k.t()) * d ** -0.5
                score[~seen] = float("-inf")
                out[first:first + new, j] = torch.nan_to_num(torch.softmax(score, -1)) @ v
        first += new
    if s["gate"] is not None:
        out = out / (1 + torch.exp(-s["gate"].double()))
    return out

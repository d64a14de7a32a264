"""The attention operators between the projections, as cases that can be timed and compared.

A Qwen3.5 engine runs, for each attention layer, the q / k / v projections, then
``rotate`` (RMS norm and multi-axis rotary of the queries), ``kv_append`` (the
same of the keys, and both into the paged cache), ``prefix_attention`` (the new
tokens over the shared prefix and their own pages) and the output projection.
``own`` false computes the three in plain torch, true calls the library.

The paged cache of both forms is the library's: a page of ``page`` tokens holds,
for each key/value head, keys as [page / 32][D / 8][32 tokens][8 columns] and
values as [page / 8][D][8 tokens].  Token j of a sequence whose page list is p
lies in slot p[j // page] * page + j % page.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
EPS = 1e-6
E4M3_MAX = 448.0


# ---- the cases ---------------------------------------------------------------------------------------------------

def listed() -> list[dict]:
    return [
        # one decoded token's queries, out of the gated q projection (each head's 256 queries, then its 256 gates)
        _rotate("rotate_b1", 1, 16, 256, 64, [11, 11, 10], True, "f32", "f16", gated=True, norm=True),
        # a prefill chunk with an image in it: positions differ by axis
        _rotate("rotate_image_chunk", 251, 16, 256, 64, [11, 11, 10], True, "f32", "f16", gated=True, norm=True),
        # a long prompt of a model that rotates whole heads, one axis, bf16 activations
        _rotate("rotate_long", 8192, 32, 128, 128, [], False, "bf16", "bf16", gated=False, norm=False),
        # one decode step of eight sequences
        _append("append_b8", 8, 4, 256, 64, [11, 11, 10], True, "f32", "f16", page=64, norm=True),
        # a prefill chunk's odd remainder into an 8-bit cache
        _append("append_chunk_e4m3", 249, 4, 256, 64, [11, 11, 10], True, "f32", "e4m3", page=128, norm=True),
        # a long prompt, sections in a row, bf16 in and out
        _append("append_long", 8192, 8, 128, 128, [16, 24, 24], False, "bf16", "bf16", page=256, norm=False),
        # one sequence, early in its answer, no shared prefix: latency
        _attend("decode_b1_short", 1, [1], 0, [517], 16, 4, 256, "f16", "f16", page=64, gate="f32"),
        # eight sequences after one system prompt
        _attend("decode_b8_prefix", 8, [1], 8191, [37, 600, 1, 255, 130, 512, 33, 64], 16, 4, 256, "f16", "f16",
                page=64, gate="f32"),
        # five answers about one long document, 8-bit cache
        _attend("decode_b5_long_e4m3", 5, [1], 100003, [1, 2900, 800, 127, 1500], 16, 4, 256, "f16", "e4m3",
                page=256, gate="f32"),
        # a full serving batch after a shared prompt, another head layout, bf16
        _attend("decode_b64_prefix", 64, [1], 16384, [1 + (37 * s * s) % 500 for s in range(64)], 32, 8, 128, "bf16",
                "bf16", page=128, gate=""),
        # the next chunk of a prompt that continues a shared prefix
        _attend("chunk_256_prefix", 1, [256], 16001, [700], 16, 4, 256, "f16", "f16", page=256, gate="f32"),
        # drafted tokens checked under a sliding window with attention sinks
        _attend("verify_b4_window", 4, [5, 1, 9, 4], 0, [30001, 5000, 12345, 20], 16, 4, 256, "bf16", "bf16",
                page=4096, gate="", window=4096, sink=64),
    ]


def _text(numbers) -> str:
    """A case's list, as text: ``_lists`` reads it back."""
    return " ".join(str(v) for v in numbers)


def _lists(case: dict) -> dict:
    return case | {key: [int(v) for v in case[key].split()] for key in ("sections", "new", "lens") if key in case}


def _rotate(name, n, heads, dim, rot, sections, interleaved, dtype, out, gated, norm):
    return {"name": name, "kind": "rotate", "n": n, "heads": heads, "dim": dim, "rot": rot, "sections": _text(sections),
            "interleaved": interleaved, "dtype": dtype, "out": out, "gated": gated, "norm": norm}


def _append(name, n, heads, dim, rot, sections, interleaved, dtype, cache, page, norm):
    return {"name": name, "kind": "append", "n": n, "heads": heads, "dim": dim, "rot": rot, "sections": _text(sections),
            "interleaved": interleaved, "dtype": dtype, "cache": cache, "page": page, "norm": norm}


def _attend(name, seqs, new, prefix, lens, heads, kv_heads, dim, dtype, cache, page, gate, window=0, sink=0):
    """Per sequence ``new`` new tokens, ``lens`` own ones (the new ones among them), after ``prefix`` shared ones."""
    new = new * seqs if len(new) == 1 else new
    return {"name": name, "kind": "attend", "new": _text(new), "prefix": prefix, "lens": _text(lens),
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "cache": cache, "page": page,
            "gate": gate, "window": window, "sink": sink}


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["rotate", "append", "attend", "attend"])
    dim = rng.choice([64, 128, 256])
    flip = lambda: rng.random() < 0.5  # noqa: E731
    if kind != "attend":
        rot = rng.choice([dim, dim // 2, dim // 4])
        interleaved = flip()
        third = rot // 2 // 3
        sections = rng.choice([[], [rot // 2 - 2 * third, third, third]])
        n, heads = _log_int(rng, 1, 8192), rng.randint(1, 32)
        if kind == "append":
            heads = rng.choice([1, 2, 3, 4, 8])
            c = _append("", n, heads, dim, rot, sections, interleaved, rng.choice(["f32", "f16", "bf16"]),
                        rng.choice(["f16", "bf16", "e4m3"]), rng.choice([32, 64, 96, 256, 4096]), flip())
        else:
            c = _rotate("", n, heads, dim, rot, sections, interleaved, *rng.choice([
                ("f32", "f16"), ("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16")]), flip(), flip())
    else:
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 6, 8])
        seqs = _log_int(rng, 1, 64)
        most = _log_int(rng, 1, max(1, 256 // seqs)) if flip() else 1
        new = [rng.randint(1, most) for _ in range(seqs)]
        prefix = _log_int(rng, 1, 100000) if rng.random() < 0.7 else 0
        top = _log_int(rng, most, 4096 if prefix else 32768)
        lens = [max(k, _log_int(rng, 1, top)) for k in new]
        cache = rng.choice(["f16", "bf16", "e4m3"])
        dtype = cache if cache != "e4m3" else rng.choice(["f16", "bf16"])
        window, sink = (_log_int(rng, 16, 8192), rng.choice([0, 4, 64])) if rng.random() < 0.25 else (0, 0)
        page = rng.choice([32, 64, 96, 256, 4096])
        c = _attend("", seqs, new, prefix, lens, heads, kv_heads, dim, dtype, cache, page,
                    rng.choice(["", "f32", dtype]), window, sink)
        flops, size = (max(work(x)[key] for x in listed()) for key in ("flops", "bytes"))
        while (work(c)["flops"] > flops or work(c)["bytes"] > size or seqs * max(lens) * kv_heads * dim > 1 << 28
               or seqs * max(new) * heads * (c["prefix"] + max(lens)) > 1 << 29):  # (what the plain form holds)
            lens = [max(k, v // 2) for k, v in zip(new, lens)]
            c |= {"prefix": c["prefix"] // 2, "lens": _text(lens)}
    del c["name"]
    return c


def work(case: dict) -> dict:
    c = _lists(case)
    if c["kind"] == "rotate":
        n = c["n"] * c["heads"] * c["dim"]
        axes = len(c["sections"]) or 1
        return {"bytes": n * (SIZE[c["dtype"]] + SIZE[c["out"]]) + 4 * axes * c["n"],
                "flops": n * (3 * c["rot"] / c["dim"] + (4 if c["norm"] else 0))}
    if c["kind"] == "append":
        n = c["n"] * c["heads"] * c["dim"] * 2
        axes = len(c["sections"]) or 1
        return {"bytes": n * (SIZE[c["dtype"]] + SIZE[c["cache"]]) + (8 + 4 * axes) * c["n"],
                "flops": n / 2 * (3 * c["rot"] / c["dim"] + (4 if c["norm"] else 0))}
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
    return {"bytes": seen * c["kv_heads"] * 2 * c["dim"] * SIZE[c["cache"]] + rows * 2 * SIZE[c["dtype"]]
            + (rows * SIZE[c["gate"]] if c["gate"] else 0),
            "flops": 4 * c["heads"] * c["dim"] * pairs}


# ---- what a program has in hand before the call ------------------------------------------------------------------

def _generator(seed: int) -> torch.Generator:
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _positions(g, n: int, sections: list) -> torch.Tensor:
    """A prompt's positions, far into a long context: text counts all axes together, an image of a quarter of the
    tokens keeps its time and walks its rows and columns."""
    start = torch.randint(0, 200000, (1,), generator=g, device=DEV)
    t = start + torch.arange(n, device=DEV)
    if not sections:
        return t.to(torch.int32)
    lo, hi = n // 4, n // 2
    wide = max(1, math.isqrt(max(1, hi - lo)))
    cell = torch.arange(n, device=DEV) - lo
    image = (cell >= 0) & (cell < hi - lo)
    rows = [torch.where(image, start + lo, t), torch.where(image, start + lo + cell // wide, t),
            torch.where(image, start + lo + cell % wide, t)]
    return torch.stack(rows).to(torch.int32).contiguous()


def _head_scale(g, heads: int, top: float) -> torch.Tensor:
    """Scale of an 8-bit head: its largest magnitude over the type's."""
    return (torch.rand(heads, generator=g, device=DEV) * 0.5 + 0.75) * (top / E4M3_MAX)


def prepare(case: dict, seed: int):
    c, g = _lists(case), _generator(seed)
    normal = lambda *shape: torch.randn(shape, generator=g, device=DEV)  # noqa: E731
    s: dict = {"case": c}
    if c["kind"] == "attend":
        return _prepare_attend(c, s, g)
    n, h, d = c["n"], c["heads"], c["dim"]
    s["positions"] = _positions(g, n, c["sections"])
    s["norm"] = torch.rand(d, generator=g, device=DEV) + 0.5 if c["norm"] else None
    if c["kind"] == "rotate":
        x = normal(n, h, 2 * d if c["gated"] else d).to(DTYPES[c["dtype"]])
        s["x"] = x[..., :d]
    else:
        s["k"] = normal(n, h, d).to(DTYPES[c["dtype"]])
        s["v"] = normal(n, h, d).to(DTYPES[c["dtype"]])
        page = c["page"]
        pages = (n + page - 1) // page + 2
        order = torch.randperm(pages, generator=g, device=DEV)
        at = torch.arange(n, device=DEV) + page // 2  # the prompt continues in the middle of a page
        s["slots"] = (order[at // page] * page + at % page).to(torch.int64)
        kind = DTYPES[c["cache"]]
        s["cache_k"] = normal(pages, h, page // 32, d // 8, 32, 8).to(kind)
        s["cache_v"] = normal(pages, h, page // 8, d, 8).to(kind)
        s["k_scale"] = _head_scale(g, h, 5.0) if c["cache"] == "e4m3" else None
        s["v_scale"] = _head_scale(g, h, 5.0) if c["cache"] == "e4m3" else None
    if own:  # the handles over these tensors that a program keeps
        from qwowl35_amd import attention as at_

        s["rope"] = at_.Rotary(c["rot"], 1e7, c["sections"], c["interleaved"], device=DEV)
        if c["kind"] == "append":
            s["cache"] = at_.PagedCache(s["cache_k"], s["cache_v"], s["k_scale"], s["v_scale"])
    return s


def _prepare_attend(c, s, g):
    d, page, kind = c["dim"], c["page"], DTYPES[c["cache"]]
    count = lambda n: (n + page - 1) // page  # noqa: E731
    seqs, total = len(c["new"]), sum(c["new"])
    own_pages = [count(n) for n in c["lens"]]
    pages = count(c["prefix"]) + sum(own_pages) + 1
    normal = lambda *shape: torch.randn(shape, generator=g, device=DEV)  # noqa: E731
    spread = 1.0
    if c["cache"] == "e4m3":
        s["k_scale"], s["v_scale"] = _head_scale(g, c["kv_heads"], 5.0), _head_scale(g, c["kv_heads"], 5.0)
        spread = E4M3_MAX / 5.0
    else:
        s["k_scale"] = s["v_scale"] = None
    cached = lambda *shape: normal(*shape).mul_(spread).clamp_(-E4M3_MAX, E4M3_MAX).to(kind)  # noqa: E731
    s["cache_k"] = cached(pages, c["kv_heads"], page // 32, d // 8, 32, 8)
    s["cache_v"] = cached(pages, c["kv_heads"], page // 8, d, 8)
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
    # queries that single some keys out: logits of standard deviation 2
    s["q"] = (normal(total, c["heads"], d) * 2).to(DTYPES[c["dtype"]])
    s["gate"] = None
    if c["gate"]:  # the gate half of each head of the q projection
        s["gate"] = normal(total, c["heads"], 2 * d).to(DTYPES[c["gate"]])[..., d:]
    if own:
        from qwowl35_amd import attention as at_

        s["cache"] = at_.PagedCache(s["cache_k"], s["cache_v"], s["k_scale"], s["v_scale"])
        s["workspace"] = at_.prefix_attention_workspace(s["cache"], c["heads"], seqs, total, device=DEV)
        s["max_new"] = max(c["new"])
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------

def run(s):
    c = s["case"]
    if own:
        from qwowl35_amd import attention as at_

        if c["kind"] == "rotate":
            return at_.rotate(s["x"], s["rope"], s["positions"], norm=s["norm"], eps=EPS, out_dtype=DTYPES[c["out"]])
        if c["kind"] == "append":
            at_.kv_append(s["cache"], s["k"], s["v"], s["slots"], rope=s["rope"], positions=s["positions"],
                          norm=s["norm"], eps=EPS)
            return s["cache_k"], s["cache_v"]
        return at_.prefix_attention(s["q"], s["cache"], s["pages"], s["lengths"], s["starts"],
                                    max_new=s["max_new"], prefix_pages=s["prefix_pages"], prefix_len=c["prefix"],
                                    window=c["window"], sink=c["sink"], gate=s["gate"], workspace=s["workspace"])
    if c["kind"] == "rotate":
        return _plain_rotate(c, s["x"], s["positions"], s["norm"]).to(DTYPES[c["out"]])
    if c["kind"] == "append":
        return _plain_append(c, s)
    return _plain_attend(c, s)


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


def _plain_append(c, s):
    k = _plain_rotate(c, s["k"], s["positions"], s["norm"])
    v = s["v"].float()
    if s["k_scale"] is not None:
        k = (k / s["k_scale"][:, None]).clamp(-E4M3_MAX, E4M3_MAX)
        v = (v / s["v_scale"][:, None]).clamp(-E4M3_MAX, E4M3_MAX)
    page, at = s["slots"] // c["page"], s["slots"] % c["page"]
    kind, n, h, d = DTYPES[c["cache"]], c["n"], c["heads"], c["dim"]
    byte = torch.uint8 if c["cache"] == "e4m3" else kind  # (indexed stores take no 8-bit floats)
    k = k.to(kind).view(byte).view(n, h, d // 8, 8)
    s["cache_k"].view(byte).permute(0, 2, 4, 1, 3, 5)[page, at // 32, at % 32] = k
    s["cache_v"].view(byte).permute(0, 2, 4, 1, 3)[page, at // 8, at % 8] = v.to(kind).view(byte)
    return s["cache_k"], s["cache_v"]


def _tokens(cache_k, cache_v, pages):
    """Keys and values [..., tokens, heads, D] in float32 of pages [..., m]."""
    byte = torch.uint8 if cache_k.dtype == torch.float8_e4m3fn else cache_k.dtype
    k = cache_k.view(byte)[pages.long()].view(cache_k.dtype).float()  # [..., m, h, page / 32, D / 8, 32, 8]
    v = cache_v.view(byte)[pages.long()].view(cache_v.dtype).float()  # [..., m, h, page / 8, D, 8]
    k = k.movedim(-2, -3).movedim(-5, -3)                             # [..., m, page / 32, 32, h, D / 8, 8]
    v = v.movedim(-1, -2).movedim(-4, -2)                             # [..., m, page / 8, 8, h, D]
    lead, m, h, d = pages.shape[:-1], pages.shape[-1], cache_k.shape[1], cache_v.shape[3]
    page = cache_v.shape[2] * 8
    return k.reshape(*lead, m * page, h, d), v.reshape(*lead, m * page, h, d)


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
    pk, pv = _tokens(s["cache_k"], s["cache_v"], s["prefix_pages"])
    ok, ov = _tokens(s["cache_k"], s["cache_v"], s["pages"])
    pk, pv, ok, ov = pk[:p], pv[:p], ok[:, :longest], ov[:, :longest]
    if s["k_scale"] is not None:
        pk, pv = pk * s["k_scale"][:, None], pv * s["v_scale"][:, None]
        ok, ov = ok * s["k_scale"][:, None], ov * s["v_scale"][:, None]
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


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    c = s["case"]
    if c["kind"] == "rotate":
        return _exact_rotate(c, s["x"], s["positions"], s["norm"])
    if c["kind"] == "append":
        return _exact_append(c, s)
    return _exact_attend(c, s)


def _slot_index(page, heads, d, slots):
    """Flat cache index of every (slot, head, column): of keys, and of values."""
    col = torch.arange(d, device=DEV)
    head = torch.arange(heads, device=DEV)[:, None]
    slots = slots.long()[:, None, None]
    base, t = ((slots // page) * heads + head) * page * d, slots % page
    k = base + (t // 32) * 32 * d + (col // 8) * 256 + (t % 32) * 8 + col % 8
    v = base + (t // 8) * 8 * d + col * 8 + t % 8
    return k, v


def _exact_append(c, s):
    k, v = _exact_rotate(c, s["k"], s["positions"], s["norm"]), s["v"].double()
    if s["k_scale"] is not None:
        k = (k / s["k_scale"].double()[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
        v = (v / s["v_scale"].double()[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
    ck, cv = s["cache_k"].double(), s["cache_v"].double()
    ik, iv = _slot_index(c["page"], c["heads"], c["dim"], s["slots"])
    ck.view(-1)[ik.reshape(-1)] = k.reshape(-1)
    cv.view(-1)[iv.reshape(-1)] = v.reshape(-1)
    return ck, cv


def _exact_attend(c, s):
    """Sequence by sequence: its tokens' keys and values as one list, each new token's softmax over what it sees."""
    group, d, page = c["heads"] // c["kv_heads"], c["dim"], c["page"]
    byte = torch.uint8 if c["cache"] == "e4m3" else DTYPES[c["cache"]]

    def slots(pages, n):
        t = torch.arange(n, device=DEV)
        return pages.long()[t // page] * page + t % page if n else t

    def read(at):
        ik, iv = _slot_index(page, c["kv_heads"], d, at)
        k = s["cache_k"].view(byte).view(-1)[ik].view(DTYPES[c["cache"]]).double().transpose(0, 1)
        v = s["cache_v"].view(byte).view(-1)[iv].view(DTYPES[c["cache"]]).double().transpose(0, 1)
        if s["k_scale"] is not None:
            k, v = k * s["k_scale"].double()[:, None, None], v * s["v_scale"].double()[:, None, None]
        return k, v  # [kv head, tokens, d]

    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    prefix = read(slots(s["prefix_pages"], c["prefix"]))
    first = 0
    for i, (new, length) in enumerate(zip(c["new"], c["lens"])):
        mine = read(slots(s["pages"][i], length))
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

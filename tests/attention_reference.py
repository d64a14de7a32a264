"""The attention operators' formulas in float64 on the CPU, with the bounds that
their kernels' roundings give, for the tests."""
from __future__ import annotations

import math

import torch

EPS = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8,
       torch.float8_e4m3fn: 2.0 ** -4}  # half a step, relative
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0,
        torch.float8_e4m3fn: 2.0 ** -10}  # half a subnormal step


def rotate(x, rot, base, positions, sections=(), interleaved=False, norm=None, eps=1e-6):
    """(rotated rows, bound of the fp32 arithmetic) of x [n, heads, dim]; positions [n] or [axes, n]."""
    x = x.double().cpu()
    if norm is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * norm.double().cpu()
    y, bound = x.clone(), x.abs().clone()
    if rot:
        half = rot // 2
        positions = positions.double().cpu()
        ends = torch.tensor(list(sections)).cumsum(0).tolist() if sections else []
        for i in range(half):
            if not sections or positions.dim() == 1:
                at = positions if positions.dim() == 1 else positions[0]
            elif interleaved:
                axis = i % 3
                at = positions[axis if axis and i < 3 * sections[axis] else 0]
            else:
                at = positions[next(k for k, e in enumerate(ends) if i < e)]
            angle = (at * base ** (-2.0 * i / rot))[:, None]
            a, b = x[..., i], x[..., i + half]
            y[..., i] = a * angle.cos() - b * angle.sin()
            y[..., i + half] = b * angle.cos() + a * angle.sin()
            bound[..., i] = bound[..., i + half] = a.abs() + b.abs()
    # sine and cosine within 2 steps and an angle 2^-25 of half a turn off (pi 2^-25 < 2 steps), the norm's mean,
    # root, quotient and two products, and the rotation's two products and sum: under 16 half steps of fp32
    return y, bound * 16 * 2.0 ** -24


def close(got, want, bound, what=""):
    """|got - want| within `bound` plus half a step of got's type."""
    got, t = got.cpu(), got.dtype
    got = got.double() if t != torch.float8_e4m3fn else got.float().double()
    limit = bound * (1 + EPS[t]) + want.abs() * EPS[t] + TINY[t]
    off = (got - want).abs()
    bad = ~(off <= limit)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} values off, the worst "
                           f"{float((off / limit.clamp_min(1e-300))[bad].max()):.3g} of its bound")


def pack(cache, slots, k, v):
    """Puts tokens [n, heads, dim] (any float type) into a PagedCache's slots by the documented layout."""
    d, page = cache.head_dim, cache.page_size
    byte = torch.uint8 if cache.k.dtype == torch.float8_e4m3fn else cache.k.dtype
    slots = slots.to(cache.k.device)
    pg, at = slots // page, slots % page
    n, h = k.shape[:2]
    cache.k.view(byte).permute(0, 2, 4, 1, 3, 5)[pg, at // 32, at % 32] = \
        k.to(cache.k.device).to(cache.k.dtype).view(byte).view(n, h, d // 8, 8)
    cache.v.view(byte).permute(0, 2, 4, 1, 3)[pg, at // 8, at % 8] = \
        v.to(cache.k.device).to(cache.k.dtype).view(byte)


def unpack(cache, slots):
    """Tokens [n, heads, dim] as the cache's type holds them (without scales), on the CPU."""
    byte = torch.uint8 if cache.k.dtype == torch.float8_e4m3fn else cache.k.dtype
    slots = slots.to(cache.k.device)
    pg, at = slots // cache.page_size, slots % cache.page_size
    k = cache.k.view(byte).permute(0, 2, 4, 1, 3, 5)[pg, at // 32, at % 32].contiguous().view(cache.k.dtype)
    v = cache.v.view(byte).permute(0, 2, 4, 1, 3)[pg, at // 8, at % 8].contiguous().view(cache.k.dtype)
    return k.flatten(2).cpu(), v.cpu()


def attend(q, k, v, seen, scale, prob):
    """(out, bound) of one sequence: q [new, heads, dim], k and v [tokens, kv heads, dim], seen [new, tokens] bool.

    ``prob``: the 16-bit type that the kernel rounds probabilities to."""
    q, k, v = (t.double().cpu() for t in (q, k, v))
    new, heads, dim = q.shape
    group = heads // k.shape[1]
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    if k.shape[0] == 0 or new == 0:
        return out, bound
    for h in range(heads):
        kh, vh = k[:, h // group], v[:, h // group]
        s = (q[:, h] @ kh.t()) * scale
        # fp32 sums of dim products, and the scaling: each logit off by at most this
        off = float((q[:, h].abs() @ kh.abs().nan_to_num(0, 0, 0).t()).max()) * abs(scale) * (dim + 4) * 2.0 ** -24
        s = s.masked_fill(~seen, -math.inf)
        p = torch.softmax(s, -1).nan_to_num(0.0)
        for j in range(new):  # (row by row: a value that a row does not see is no part of its sum)
            w = seen[j]
            pj, vj = p[j][w], vh[w]
            out[j, h] = pj @ vj
            top = float(vj.abs().max()) if vj.numel() else 0.0
            # probabilities: rounded to `prob` (in its subnormals by half a step of those, against a sum of at
            # least one), exponentials and rescalings to 2^-18, and twice the logits' error
            bound[j, h] = (EPS[prob] + 2.0 ** -18 + 2 * off) * (pj @ vj.abs()) + TINY[prob] * int(w.sum()) * top
    return out, bound

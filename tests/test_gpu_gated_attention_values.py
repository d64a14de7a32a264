"""The layer against its formulas in float64, step by step, so that each step has
its own operator's bound: the library's projections, the queries' rotation, what
the cache holds, the attention over that, and the output projection."""
from __future__ import annotations

import pytest
import torch

from tests import attention_reference as ref
from tests.test_gpu_gated_attention import DIM, E, HEADS, KV, ROT, SECTIONS, _layer

pytestmark = pytest.mark.gpu


def _product(layer, name, x, dst=None):
    """The library's product, by the kernel that the layer takes for as many tokens."""
    from qwowl35_amd import _ffi
    from qwowl35_amd import runtime as rt

    w = layer.weights[name]
    if x.shape[0] <= _ffi.MAX_BATCH:
        return rt.decode_matvec(w, x, dst=dst, residual=dst is not None)
    return rt.matmul_prefill(w.prefill, x, out_dtype=torch.float32, dst=dst,
                             epilogue=_ffi.EPILOGUE_STORE if dst is None else _ffi.EPILOGUE_ADD)


def _check(layer, x, residual, positions, slots, own, lens, new, prefix, window, sink, turned, core, got):
    """A call: ``own`` each sequence's slots, ``lens`` its tokens after it; ``turned`` and ``core`` are the layer's."""
    c, n = layer.cache, x.shape[0]
    q, k, v = (_product(layer, f"attn_{p}", x).view(n, h, -1) for p, h in (("q", HEADS), ("k", KV), ("v", KV)))
    turn = lambda t, norm: ref.rotate(t, ROT, 1e6, positions, SECTIONS, True, norm)  # noqa: E731
    ref.close(turned, *turn(q[..., :DIM], layer.q_norm), "queries")
    scales = [torch.ones(KV, 1, dtype=torch.float64) if s is None else s.double().cpu()[:, None]
              for s in (c.k_scale, c.v_scale)]
    top = 448.0 if c.k_scale is not None else float("inf")
    gk, gv = ref.unpack(c, slots.cpu())
    wk, bk = turn(k, layer.k_norm)
    for what, cached, want, bound, s in (("keys", gk, wk, bk, scales[0]), ("values", gv, v.double().cpu(), 0.0, scales[1])):
        want = (want / s).clamp(-top, top)
        ref.close(cached, want, bound / s + want.abs() * 2.0 ** -23, what)
    wants, bounds, first = [], [], 0
    for s, (length, m) in enumerate(zip(lens, new)):
        at = torch.cat([prefix, own[s][:length]]).cpu()
        kk, vv = (t.float().double() * f for t, f in zip(ref.unpack(c, at), scales))
        where, p = torch.arange(len(at)), len(at) - m + torch.arange(m)[:, None]
        seen = where <= p
        if window:
            seen &= (where > p - window) | (where < sink)
        o, b = ref.attend(turned[first:first + m], kk, vv, seen, DIM ** -0.5, layer.q_dtype)
        wants.append(o), bounds.append(b)
        first += m
    want, bound = torch.cat(wants), torch.cat(bounds)
    if layer.gated:
        g = torch.sigmoid(q[..., DIM:].double().cpu())
        want, bound = want * g, bound * g + (want * g).abs() * 2.0 ** -20
    assert core.dtype == torch.float32
    ref.close(core.view(n, HEADS, DIM), want, bound, "attention")
    assert torch.equal(got, _product(layer, "attn_output", core.reshape(n, -1), residual.clone()))


@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("cache_dtype", [torch.float16, torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("window,sink", [(0, 0), (33, 4)])
def test_every_step_of_the_layer(cuda, gated, cache_dtype, window, sink, monkeypatch):
    """A prompt, then two sequences that continue it by chunks and single tokens."""
    from qwowl35_amd import attention as at_

    layer, rand = _layer(cuda, gated, cache_dtype)
    layer.window, layer.sink = window, sink
    made = []
    for name in ("rotate", "prefix_attention"):
        monkeypatch.setattr(at_, name, lambda *a, run=getattr(at_, name), **k: (made.append(run(*a, **k)), made[-1])[1])
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    axes = lambda p: torch.stack([p, p // 2, p % 7]).to(torch.int32).contiguous()  # noqa: E731
    shared, pages = i32([7, 2]), i32([[0, 5], [9, 4]])
    n = torch.arange(40, device=cuda)
    prefix = layer.cache.slots(shared, n)

    def step(x, pos, slots, own, lens, new, before, **kw):
        residual = rand(*x.shape)
        got = residual.clone()
        made.clear()
        starts = i32([0] + torch.tensor(new).cumsum(0).tolist())
        layer(x, got, pos, slots, kw.pop("pages"), i32(lens), starts, **kw)
        assert len(made) == 2
        _check(layer, x, residual, pos, slots, own, lens, new, before, window, sink, *made, got)

    step(rand(40, E), axes(n), prefix, [prefix], [40], [40], prefix[:0], pages=shared.view(1, 2))
    own = [layer.cache.slots(p, torch.arange(64, device=cuda)) for p in pages]
    done = [0, 0]
    for new in ([5, 3], [1, 1], [30, 12], [1, 4]):
        at = [torch.arange(d, d + m, device=cuda) for d, m in zip(done, new)]
        done = [d + m for d, m in zip(done, new)]
        step(rand(sum(new), E), axes(torch.cat([a + 40 for a in at])), torch.cat([own[s][a] for s, a in enumerate(at)]), own,
             done, new, prefix, pages=pages, max_new=max(new), prefix_pages=shared, prefix_len=40)

"""The block-scaled cache as a program uses it: in an attention layer with its
projections, on other streams and devices than the current ones, in calls that
overlap."""
from __future__ import annotations

import pytest
import torch

from tests import attention_reference as ref
from tests.block_reference import BlockBatch, close
from tests.test_gpu_attention import BF16, E4M3, F16, F32, _gen
from tests.test_gpu_attention_devices import elsewhere  # noqa: F401
from tests.test_gpu_gated_attention import DIM, E, HEADS, KV, PAGE, ROT, SECTIONS, _layer
from tests.test_gpu_streams import _busy, _made_on

pytestmark = pytest.mark.gpu

I8 = torch.int8


def _over(layer, kind, cuda):
    """The layer over a block-scaled cache."""
    from qwowl35_amd import attention as at

    cache = at.PagedCache.empty(10, KV, PAGE, DIM, kind, device=cuda, block_scales=True)
    return at.GatedAttention(layer.weights, cache, HEADS, layer.rope, q_norm=layer.q_norm, k_norm=layer.k_norm, max_seqs=4,
                             max_tokens=layer.max_tokens)


@pytest.mark.parametrize("kind", [I8, E4M3])
def test_a_layer_from_prompt_to_decode(cuda, kind):
    """A shared prompt, two sequences that continue it and decoded tokens: every call's attention against the formula
    over what the cache then holds, and the layer the same bits as its operators."""
    from qwowl35_amd import attention as at
    from qwowl35_amd import runtime as rt

    plain, rand = _layer(cuda, True, F16)
    layer, other = _over(plain, kind, cuda), _over(plain, kind, cuda)
    assert layer.q_dtype == F16
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    axes = lambda p: torch.stack([p, p // 2, p % 7]).to(torch.int32).contiguous()  # noqa: E731
    shared, pages, done = i32([7, 2]), i32([[0, 5], [9, 4]]), [0, 0]
    for step, new in enumerate(([40], [5, 3], [1, 1], [1, 1])):
        if step == 0:
            t = torch.arange(40, device=cuda)
            slots, positions, args = layer.cache.slots(shared, t), axes(t), (shared.view(1, 2), i32([40]), i32([0, 40]))
            kw = {}
        else:
            t = [torch.arange(d, d + n, device=cuda) for d, n in zip(done, new)]
            done = [d + n for d, n in zip(done, new)]
            slots = torch.cat([layer.cache.slots(pages[s], x) for s, x in enumerate(t)])
            positions, args = axes(torch.cat(t) + 40), (pages, i32(done), i32([0, new[0], sum(new)]))
            kw = {"max_new": max(new), "prefix_pages": shared, "prefix_len": 40}
        x = rand(sum(new), E)
        got = layer(x, torch.zeros_like(x), positions, slots, *args, **kw)
        n = sum(new)
        q, k, v = (other._project(w, x) for w in ("attn_q", "attn_k", "attn_v"))
        q, k, v = q.view(n, HEADS, -1), k.view(n, KV, DIM), v.view(n, KV, DIM)
        at.kv_append(other.cache, k, v, slots, layer.rope, positions, layer.k_norm)
        turned = at.rotate(q[..., :DIM], layer.rope, positions, layer.q_norm, out_dtype=F16)
        core = at.prefix_attention(turned, other.cache, *args, gate=q[..., DIM:], out_dtype=F32, **kw)
        want = torch.zeros_like(x)
        out = layer.weights["attn_output"]
        if n <= 8:
            rt.decode_matvec(out, core.view(n, -1), dst=want, residual=True)
        else:
            rt.matmul_prefill(out.prefill, core.view(n, -1), out_dtype=F32, dst=want, epilogue=1)
        assert torch.equal(got, want), step
        # the attention by the formula, over what the cache holds
        bare = at.prefix_attention(turned, other.cache, *args, out_dtype=F32, **kw)
        first = 0
        for s, m in enumerate(new):
            held = layer.cache.slots(shared, torch.arange(40, device=cuda))
            if step:
                held = torch.cat([held, layer.cache.slots(pages[s], torch.arange(done[s], device=cuda))])
            kk, vv = at.kv_read(layer.cache, held, dtype=F32)
            seen = torch.arange(len(held)) <= len(held) - m + torch.arange(m)[:, None]
            o, b = ref.attend(turned[first:first + m], kk, vv, seen, DIM ** -0.5, F16)
            close(bare[first:first + m], o, b * (1 + 2.0 ** -5), f"step {step}, sequence {s}")
            first += m
        # what was written is the rotated key within half a step of its block's scale
        wk, bound = ref.rotate(k, ROT, 1e6, positions, SECTIONS, True, layer.k_norm)
        back = at.kv_read(layer.cache, slots, dtype=F32)[0].double().cpu()
        scale = layer.cache.k_scale[slots // PAGE, :, slots % PAGE // 32].double().cpu()[..., None]
        half = scale / 2 if kind == I8 else torch.maximum(wk.abs() * ref.EPS[E4M3], scale * ref.TINY[E4M3])
        assert ((back - wk).abs() <= half + 2 * bound).all()


def test_on_another_stream(cuda):
    """Append and reading run behind what the current stream holds, and make what they return on theirs."""
    from qwowl35_amd import attention as at

    randn = _gen(cuda, 1)
    k, v = randn(40, 2, 64), randn(40, 2, 64)
    slots = torch.arange(40, device=cuda)
    here, there = (at.PagedCache.empty(2, 2, 32, 64, I8, device=cuda) for _ in range(2))
    at.kv_append(here, k, v, slots)
    want = at.kv_read(here, slots)
    late, side = torch.zeros_like(k), torch.cuda.Stream()
    torch.cuda.synchronize()
    _busy()
    late.copy_(k)
    at.kv_append(there, late, v, slots, stream=side)
    got = at.kv_read(there, slots, stream=side)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b) and _made_on(a) == side.cuda_stream


def test_on_another_device(cuda, elsewhere):  # noqa: F811
    from qwowl35_amd import attention as at

    x = _gen(cuda, 1)(3, 2, 64)
    cache = at.PagedCache(torch.zeros(1, 2, 1, 8, 32, 8, dtype=I8, device=cuda), torch.zeros(1, 2, 4, 64, 8, dtype=I8, device=cuda),
                          torch.zeros(1, 2, 1, device=cuda), torch.zeros(1, 2, 1, device=cuda))
    slots = torch.arange(3, device=cuda)
    at.kv_append(cache, x, x, slots)
    k, v = at.kv_read(cache, slots, dtype=F32)
    assert elsewhere == [0, 0] and torch.equal(k, v) and (k - x).abs().max() <= 2.0 ** -5


def test_calls_that_overlap(cuda):
    """Appends to blocks of their own, and attention with workspaces of their own, on three streams at a time."""
    from qwowl35_amd import attention as at

    kv, dim, heads = 2, 128, 4
    randn = _gen(cuda, 5)
    one, other = (at.PagedCache.empty(12, kv, 64, dim, I8, device=cuda) for _ in range(2))
    pages = [torch.tensor([[p, p + 1]], dtype=torch.int32, device=cuda) for p in (0, 4, 8)]
    n = 100
    at_ = torch.arange(n, device=cuda)
    slots = [one.slots(p[0], at_) for p in pages]
    k, v, q = ([randn(n, h, dim) for _ in pages] for h in (kv, kv, heads))
    q = [x.to(F16) for x in q]
    lengths, starts = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in ([n], [0, n]))

    def call(c, i):
        at.kv_append(c, k[i], v[i], slots[i])
        return at.prefix_attention(q[i], c, pages[i], lengths, starts)

    want = [call(other, i) for i in range(3)]
    streams = [torch.cuda.Stream() for _ in pages]
    torch.cuda.synchronize()
    got = []
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            _busy()
            got.append(call(one, i))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype,kind", [(F16, I8), (BF16, E4M3)])
def test_the_same_bits_every_time(cuda, dtype, kind):
    b = BlockBatch(cuda, [3, 70, 1], [300, 70, 1200], 2000, 8, 2, 256, 64, dtype, kind, seed=3)
    want = b.run()
    for _ in range(3):
        got = b.run()
        nan = want.isnan()
        assert torch.equal(got.isnan(), nan) and torch.equal(got[~nan], want[~nan])

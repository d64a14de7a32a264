"""One attention layer with its projections: a shared prompt as a prefill chunk,
two sequences that continue it, and decoded tokens, against the layer in float64
and recorded into a graph."""
from __future__ import annotations

import math

import pytest
import torch

from tests import attention_reference as ref

pytestmark = pytest.mark.gpu

E, HEADS, KV, DIM, ROT, PAGE = 256, 4, 2, 64, 32, 32
SECTIONS = [6, 5, 5]


def _layer(cuda, gated, cache_dtype, max_tokens=64):
    from qwowl35_amd import attention as at
    from qwowl35_amd import runtime as rt

    g = torch.Generator(device=cuda)
    g.manual_seed(21)
    rand = lambda *s: torch.randn(s, generator=g, device=cuda)  # noqa: E731
    rows = {"attn_q": HEADS * DIM * (2 if gated else 1), "attn_k": KV * DIM, "attn_v": KV * DIM, "attn_output": E}
    weights = {n: rt.quantize_weight(rand(r, HEADS * DIM if n == "attn_output" else E) * 0.06, rt.TYPE_Q8_0)
               for n, r in rows.items()}
    scale = {}
    if cache_dtype == torch.float8_e4m3fn:
        scale = {k: torch.full((KV,), 6.0 / 448, device=cuda) for k in ("k_scale", "v_scale")}
    cache = at.PagedCache.empty(10, KV, PAGE, DIM, cache_dtype, device=cuda, **scale)
    layer = at.GatedAttention(weights, cache, HEADS, at.Rotary(ROT, 1e6, SECTIONS, True, device=cuda),
                              q_norm=rand(DIM).abs() + 0.5, k_norm=rand(DIM).abs() + 0.5, max_seqs=4,
                              max_tokens=max_tokens)
    return layer, rand


def _want(layer, x, positions, new):
    """The layer's output for the last ``new`` of a sequence's inputs x [tokens, E], in float64 from its formulas."""
    from qwowl35_amd import runtime as rt

    w = {n: rt.dequantize(v).double().cpu().view(v.rows, v.k) for n, v in layer.weights.items()}
    x = x.double().cpu()
    n = x.shape[0]
    q = (x @ w["attn_q"].t()).view(n, HEADS, -1)
    k, v = ((x @ w[name].t()).view(n, KV, DIM) for name in ("attn_k", "attn_v"))
    turn = lambda t, norm: ref.rotate(t, ROT, 1e6, positions.cpu(), SECTIONS, True, norm)[0]  # noqa: E731
    seen = torch.ones(n, n, dtype=torch.bool).tril()[n - new:]
    out, _ = ref.attend(turn(q[..., :DIM], layer.q_norm)[n - new:], turn(k, layer.k_norm), v, seen, DIM ** -0.5,
                        torch.float16)
    if layer.gated:
        out = out * torch.sigmoid(q[n - new:, :, DIM:])
    return out.reshape(new, -1) @ w["attn_output"].t()


def _close(got, want, limit):
    err = float((got.double().cpu() - want).norm() / want.norm())
    assert err <= limit, f"relative L2 {err:.3g} over {limit:.3g}"


# Roundings that reach the result, relative: the four projections within 1e-3 (the library's bound for them); q and k
# half a step each, with the norms' near-unit rows logits of up to ~6 then move by 6 times their sum and 1e-3 each,
# and weights by twice that; v and the weights half a step each.
def _limit(cache_dtype):
    step = ref.EPS[cache_dtype]
    q = ref.EPS[torch.float16 if cache_dtype == torch.float8_e4m3fn else cache_dtype]
    return 2 * 6 * (step + q + 2e-3) + step + q + 3e-3


@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("cache_dtype", [torch.float16, torch.bfloat16, torch.float8_e4m3fn])
def test_prompt_continuations_and_decode(cuda, gated, cache_dtype):
    layer, rand = _layer(cuda, gated, cache_dtype)
    limit = _limit(cache_dtype)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    axes = lambda p: torch.stack([p, p // 2, p % 7]).to(torch.int32).contiguous()  # noqa: E731
    # the shared prompt: 40 tokens of one sequence in pages 7 and 2
    prompt, n = rand(40, E), torch.arange(40, device=cuda)
    shared = i32([7, 2])
    res = rand(40, E)
    before = res.clone()
    got = layer(prompt, res, axes(n), layer.cache.slots(shared, n), shared.view(1, 2), i32([40]), i32([0, 40]))
    assert got is res
    _close(res - before, _want(layer, prompt, axes(n), 40), limit)
    # two sequences continue it with 5 and 3 tokens, then with one each, twice
    pages = i32([[0, 5], [9, 4]])
    own = [rand(7, E), rand(5, E)]
    done = [0, 0]
    for new in ([5, 3], [1, 1], [1, 1]):
        at = [torch.arange(d, d + k, device=cuda) for d, k in zip(done, new)]
        x = torch.cat([o[a] for o, a in zip(own, at)])
        slots = torch.cat([layer.cache.slots(pages[s], a) for s, a in enumerate(at)])
        done = [d + k for d, k in zip(done, new)]
        res = torch.zeros(sum(new), E, device=cuda)
        layer(x, res, axes(torch.cat([a + 40 for a in at])), slots, pages, i32(done), i32([0, new[0], sum(new)]),
              max_new=max(new), prefix_pages=shared, prefix_len=40)
        first = 0
        for s in range(2):
            all_x, p = torch.cat([prompt, own[s][:done[s]]]), torch.arange(40 + done[s], device=cuda)
            _close(res[first:first + new[s]], _want(layer, all_x, axes(p), new[s]), limit)
            first += new[s]


def test_layer_is_its_operators(cuda):
    """The same bits as the calls one by one."""
    from qwowl35_amd import attention as at
    from qwowl35_amd import runtime as rt

    layer, rand = _layer(cuda, True, torch.float16)
    x, n = rand(3, E), torch.arange(3, device=cuda, dtype=torch.int32)
    pages, lengths = torch.tensor([[1]], dtype=torch.int32, device=cuda), torch.tensor([3], dtype=torch.int32, device=cuda)
    starts = torch.tensor([0, 3], dtype=torch.int32, device=cuda)
    slots = layer.cache.slots(pages[0], n)
    got = layer(x, torch.zeros(3, E, device=cuda), n, slots, pages, lengths, starts)
    q = rt.decode_matvec(layer.weights["attn_q"], x).view(3, HEADS, 2 * DIM)
    k, v = (rt.decode_matvec(layer.weights[w], x).view(3, KV, DIM) for w in ("attn_k", "attn_v"))
    at.kv_append(layer.cache, k, v, slots, layer.rope, n, layer.k_norm)
    core = at.prefix_attention(at.rotate(q[..., :DIM], layer.rope, n, layer.q_norm, out_dtype=torch.float16), layer.cache,
                               pages, lengths, starts, gate=q[..., DIM:], out_dtype=torch.float32)
    assert torch.equal(got, rt.decode_matvec(layer.weights["attn_output"], core.view(3, -1)))


def test_recorded_decode_steps(cuda):
    """A captured decode step of two sequences, replayed with eager work between, against eager steps."""
    layer, rand = _layer(cuda, True, torch.float16, max_tokens=8)
    other, _ = _layer(cuda, True, torch.float16, max_tokens=8)
    pages = torch.tensor([[3, 1], [8, 6]], dtype=torch.int32, device=cuda)
    x, res = torch.zeros(2, E, device=cuda), torch.zeros(2, E, device=cuda)
    positions, slots = torch.zeros(2, dtype=torch.int32, device=cuda), torch.full((2,), -1, device=cuda)
    lengths = torch.ones(2, dtype=torch.int32, device=cuda)
    for t in (layer.cache, other.cache):
        t.k.zero_(), t.v.zero_()

    def step(it=layer):
        it(x, res, positions, slots, pages, lengths, max_new=1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(36):
        x.copy_(rand(2, E))
        positions.fill_(i)
        lengths.fill_(i + 1)
        at = torch.tensor(i, device=cuda)
        slots.copy_(torch.stack([layer.cache.slots(pages[s], at) for s in range(2)]))
        res.zero_()
        graph.replay()
        got = res.clone()
        res.zero_()
        step(other)
        assert torch.equal(got, res), f"step {i}"
        assert math.isfinite(float(got.abs().max()))


def test_refusals(cuda):
    from qwowl35_amd import Qw35Error
    from qwowl35_amd import attention as at

    layer, rand = _layer(cuda, True, torch.float16, max_tokens=8)
    one = torch.zeros(1, dtype=torch.int32, device=cuda)
    with pytest.raises(Qw35Error, match="over the layer's 8"):
        layer(rand(9, E), rand(9, E), one, one, one.view(1, 1), one)
    with pytest.raises(Qw35Error, match="residual must be"):
        layer(rand(1, E), rand(1, E + 1), one, one.long(), one.view(1, 1), one)
    with pytest.raises(Qw35Error, match="rows for 5 heads"):
        at.GatedAttention(layer.weights, layer.cache, 5, None)

"""Calls with a ``stream`` argument other than the current stream: what a call
makes for itself is made on the stream that it runs on."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _busy():
    """Some milliseconds of work on the current stream."""
    a = torch.ones(4096, 4096, dtype=torch.float16, device="cuda")
    for _ in range(40):
        a = torch.mm(a, a)


def _made_on(t: torch.Tensor) -> int:
    """The stream whose memory a tensor lies in."""
    at = t.data_ptr()
    return next(s["stream"] for s in torch.cuda.memory_snapshot() if s["address"] <= at < s["address"] + s["total_size"])


@pytest.fixture
def weight(cuda):
    from qwowl35_amd import runtime as rt

    g = torch.Generator(device=cuda)
    g.manual_seed(3)
    return rt.quantize_weight(torch.randn(512, 1024, generator=g, device=cuda) * 0.05, rt.TYPE_Q8_0)


def test_a_product_is_not_cleared_after_it_is_made(cuda, weight):
    """Behind work on the current stream the product's own fill would come after it."""
    from qwowl35_amd import runtime as rt

    x = torch.randn(3, 1024, device=cuda)
    want = rt.decode_matvec(weight, x)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    _busy()
    got = rt.decode_matvec(weight, x, stream=side)
    torch.cuda.synchronize()
    assert want.any() and torch.equal(got, want)


def test_results_and_workspaces_are_the_streams(cuda, weight, monkeypatch):
    from qwowl35_amd import runtime as rt

    side = torch.cuda.Stream()
    x, many, rows = (torch.randn(n, 1024, device=cuda) for n in (3, 20, 512))
    calls = {
        "matvec": lambda s: rt.decode_matvec(weight, x, stream=s),
        "swiglu": lambda s: rt.ffn_gate_up_swiglu(weight, weight, x, stream=s),
        "argmax": lambda s: rt.output_argmax(weight, x, stream=s)[0],
        "argmax logit": lambda s: rt.output_argmax(weight, x, stream=s)[1],
        "prefill": lambda s: rt.matmul_prefill(weight, many, stream=s),
        "batch": lambda s: rt.matvec_batch(weight, many, stream=s),
        "dequantize": lambda s: rt.dequantize(weight, stream=s),
        "image": lambda s: rt.prefill_image(weight, stream=s).storage,
        "quantize": lambda s: rt.quantize(rows, rt.TYPE_Q8_0, stream=s),
        "read": lambda s: rt.stream_read(rows, stream=s),
    }
    makers, make = [], torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **k: (makers.append(torch.cuda.current_stream().cuda_stream),
                                                         make(*a, **k))[1])
    for name, call in calls.items():
        want = call(None).clone()
        side.wait_stream(torch.cuda.current_stream())
        makers.clear()
        got = call(side)
        torch.cuda.synchronize()
        assert _made_on(got) == side.cuda_stream, name
        assert all(m == side.cuda_stream for m in makers), name  # (workspaces among them)
        assert torch.equal(got, want), name


def test_an_image_of_the_first_use_is_made_on_the_stream(cuda):
    """A k-quant's fp16 image that a first chunk needs, with other work on the current stream."""
    from qwowl35_amd import runtime as rt

    w = rt.quantize_weight(torch.randn(512, 1024, device=cuda) * 0.05, rt.TYPE_Q6_K)
    x = torch.randn(20, 1024, device=cuda)
    want = rt.matvec_batch(w, x)
    del w._prefill
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    _busy()
    got = rt.matvec_batch(w, x, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(got, want)

"""The attention operators work on their tensors' device, whichever is the current one."""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_attention import F16, Batch, _cache, _gen
from tests.test_gpu_gated_attention import E, _layer

pytestmark = pytest.mark.gpu


@pytest.fixture
def elsewhere(monkeypatch):
    """Another device as the current one, as far as the library sees; the devices that it makes the current one."""
    entered, current = [], [1]

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            entered.append(self.index)
            current.append(self.index)

        def __exit__(self, *_):
            current.pop()

    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[-1])
    monkeypatch.setattr(torch.cuda, "device", Device)
    return entered


def test_rotate_and_append(cuda, elsewhere):
    from qwowl35_amd import attention as at

    x = _gen(cuda, 1)(3, 2, 64)
    assert torch.equal(at.rotate(x, None), x) and elsewhere == [0]
    cache = _cache(cuda, 1, 2, 32, 64, F16)
    at.kv_append(cache, x, x, torch.arange(3, device=cuda))
    assert elsewhere == [0, 0]
    assert torch.equal(cache.v[0, :, 0, :, :3], x.permute(1, 2, 0).to(F16))


def test_attention(cuda, elsewhere, monkeypatch):
    b = Batch(cuda, [1, 2], [33, 64], 20, 4, 2, 64, 32, F16, F16, seed=12)
    got = b.run()
    assert elsewhere == [0]
    monkeypatch.undo()
    assert torch.equal(got, b.run())


def test_layer(cuda, monkeypatch, request):
    layer, rand = _layer(cuda, True, F16)
    x, n = rand(2, E), torch.arange(2, device=cuda, dtype=torch.int32)
    pages, lengths, starts = (torch.tensor(v, dtype=torch.int32, device=cuda) for v in ([[1]], [2], [0, 2]))
    slots = layer.cache.slots(pages[0], n)
    want = layer(x, torch.zeros_like(x), n, slots, pages, lengths, starts)
    entered = request.getfixturevalue("elsewhere")
    got = layer(x, torch.zeros_like(x), n, slots, pages, lengths, starts)
    assert entered == [0] and torch.equal(got, want)


def test_tensors_on_other_devices_are_refused(cuda):
    from qwowl35_amd import Qw35Error

    layer, rand = _layer(cuda, True, F16)
    x, n = rand(1, E), torch.zeros(1, device=cuda, dtype=torch.int32)
    with pytest.raises(Qw35Error, match="x must be on the cache's cuda:0, got cpu"):
        layer(x.cpu(), x.cpu(), n, n.long(), n.view(1, 1), n)
    with pytest.raises(Qw35Error, match="residual must be a contiguous fp32 .* on cuda:0"):
        layer(x, x.cpu(), n, n.long(), n.view(1, 1), n)

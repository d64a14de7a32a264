"""Arguments that the Python layer refuses before a call, over device tensors."""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_attention import F16, Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [{"window": 1 << 32}, {"sink": 1 << 40}, {"max_new": 1 << 33}, {"scale": 1e39},
                                {"prefix_len": 1 << 32}, {"window": 0.5}])
def test_numbers_past_their_types_are_the_librarys_errors(cuda, kw):
    from qwowl35_amd import Qw35Error

    b = Batch(cuda, [1], [5], 40, 2, 1, 64, 32, F16, F16)
    with pytest.raises(Qw35Error, match="out of range"):
        b.run(**kw)
    with pytest.raises(Qw35Error, match="cannot be negative"):
        b.run(window=-1)


def test_a_stream_of_another_device_is_refused(cuda):
    import types

    from qwowl35_amd import Qw35Error

    b = Batch(cuda, [1], [5], 0, 2, 1, 64, 32, F16, F16)
    with pytest.raises(Qw35Error, match="the stream is on cuda:1, the input on cuda:0"):
        b.run(stream=types.SimpleNamespace(device=torch.device("cuda", 1)))

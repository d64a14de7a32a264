"""Forms of the attention kernels that only long or large calls take."""
from __future__ import annotations

import pytest
import torch

from tests import attention_reference as ref
from tests.test_gpu_attention import F16, Batch

pytestmark = pytest.mark.gpu


def test_as_many_sequences_as_the_list_holds(cuda):
    """1580 sequences of a token each: with starts their row tiles are counted by an upper bound, which is refused."""
    from qwowl35_amd import Qw35Error

    b = Batch(cuda, [1] * 1580, [1 + s % 37 for s in range(1580)], 40, 2, 1, 256, 32, F16, F16, seed=1)
    want, bound = b.want()
    with pytest.raises(Qw35Error, match="row tiles in a call"):
        b.run()
    b.starts = None
    ref.close(b.run(), want, bound, "a token each")

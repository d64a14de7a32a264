"""No attention kernel keeps registers in scratch memory (its accumulators and
queries fill most of a wave's registers; one moved through memory in every tile
cost 840 us where 114 are enough, 256 new tokens over 16000)."""
from __future__ import annotations

from qwowl35_amd import build
from tests.test_kernel_resources import _kernels


def test_no_attention_kernel_spills_registers():
    kernels = [k for k in _kernels(build.LIB.read_bytes())
               if any(n in k[".name"] for n in ("prefix_attention", "rotate_kernel", "kv_append"))]
    main = [k for k in kernels if "prefix_attention_kernel" in k[".name"]]
    assert len(main) == 24  # three head sizes, two query types, two cache widths, with and without shared tiles
    spilled = {k[".name"]: k[".vgpr_spill_count"] for k in kernels if k[".vgpr_spill_count"]}
    assert not spilled, spilled
    # one wave a SIMD of 256 columns, two of less
    for k in main:
        assert k[".vgpr_count"] <= (512 if "ILi256E" in k[".name"] else 256), k[".name"]

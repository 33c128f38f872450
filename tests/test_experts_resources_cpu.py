"""Register budget of the expert and 4-bit kernels, checked at compile time
(CPU only): none of them spills to scratch memory, and the 256 x 256 grouped
products keep two waves per SIMD."""
from __future__ import annotations

import concurrent.futures as cf
import tempfile

import pytest

from test_resource_usage_cpu import _hipcc, _kernels, _report

SOURCES = ["grouped_bf16.hip", "grouped_f16.hip", "grouped32.hip", "q4.hip", "experts.hip"]


@pytest.mark.skipif(_hipcc() is None, reason="hipcc not available")
def test_expert_kernels_do_not_spill():
    with tempfile.TemporaryDirectory() as d:
        with cf.ThreadPoolExecutor(max_workers=len(SOURCES)) as ex:
            seen = [k for r in ex.map(lambda s: _report(s, d), SOURCES) for k in _kernels(r)]
    names = " ".join(k[0] for k in seen)
    for want in ("gemm16nt_pp_kernel", "gemm16mid_kernel", "gemm32dma_kernel", "gemm32small_kernel", "q4_kernel",
                 "route_kernel", "combine_kernel"):
        assert want in names, "no %s instantiation found in the report" % want
    spilled = [k for k in seen if k[2] > 0]
    assert not spilled, "kernels using scratch (name, VGPRs, bytes/lane): %s" % spilled
    assert all(k[1] <= 256 for k in seen if "pp_kernel" in k[0])

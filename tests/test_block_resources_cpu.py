"""Register budget of the causal block's kernels, checked at compile time (CPU
only): none of them spills to scratch memory (the windowed attention's loads in
flight could not survive it), and each keeps the waves that its layout takes."""
from __future__ import annotations

import concurrent.futures as cf
import tempfile

import pytest

from test_resource_usage_cpu import _hipcc, _kernels, _report

SOURCES = ["attention_window.hip", "attention_window_bwd.hip", "qknorm.hip", "gated_bf16.hip", "gated_f16.hip",
           "gated.hip"]


@pytest.mark.skipif(_hipcc() is None, reason="hipcc not available")
def test_block_kernels_do_not_spill():
    with tempfile.TemporaryDirectory() as d:
        with cf.ThreadPoolExecutor(max_workers=len(SOURCES)) as ex:
            seen = [k for r in ex.map(lambda s: _report(s, d), SOURCES) for k in _kernels(r)]
    names = " ".join(k[0] for k in seen)
    for want in ("win_attn_kernel", "win_split_kernel", "win_merge_kernel", "win_dq_kernel", "win_dkv_kernel",
                 "win_dkv_merge_kernel", "qk_norm_rope_kernel", "qk_norm_rope_backward_kernel", "qk_norm_sums_kernel",
                 "gemm16nt_pp_kernel", "gemm16mid_kernel", "skinny"):
        assert want in names, "no %s instantiation found in the report" % want
    spilled = [k for k in seen if k[2] > 0]
    assert not spilled, "kernels using scratch (name, VGPRs, bytes/lane): %s" % spilled
    # two waves a SIMD: two workgroups of four waves a CU, or one of eight
    assert all(k[1] <= 256 for k in seen if "win_" in k[0] or "pp_kernel" in k[0])

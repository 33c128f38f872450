"""Gated layers large enough for the 256 x 256 tiles, with what they launch on
256 CUs; shared by the host's and the GPU's tests."""
from __future__ import annotations

import ctypes
import os

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
I64, P = ctypes.c_int64, ctypes.c_void_p

# dtype, M, K, F, launches
LARGE = [
    ("bfloat16", 1419, 640, 5209, "gated 256x256"),                         # one part round, ragged both ways, odd rows of y
    ("float16", 1280, 1024, 6000, "gated 256x256"),                         # whole rows, 16-byte stores
    ("float16", 2853, 1024, 5013, "gated 256x256"),                         # a round and most of another
    ("bfloat16", 1419, 1024, 5471, "gated 256x256, 2 quartered"),
    ("float16", 1313, 1024, 5995, "gated 256x256, 26 quartered"),           # quarters past the last row
    ("bfloat16", 2691, 1024, 5995, "gated 256x256 persistent, 5 quartered"),
    ("float16", 3857, 1024, 4030, "gated 256x256 persistent"),
]

# What the sizes of test_gated_gpu.py's CASES launch, in its order.
SMALL = ["gated 16x32"] * 4 + ["gated 32x64"] * 4 + ["gated 64x64", "gated 128x128", "gated 64x64", "gated 128x128",
         "gated 128x128"] + ["gated 64x64 staged"] * 4 + ["gated 128x128 staged", "gated fp32 16 rows"] + [
         "gated fp32 product, then gate"] * 2


def plan(dtype, M, K, F, x=4096, W=4096):
    so = ctypes.CDLL(os.path.join(ROOT, "scaffolding_amd", "libsfgemm.so"))
    buf = ctypes.create_string_buffer(96)
    code = {"float32": 0, "float16": 1, "bfloat16": 2}[dtype]
    assert so.sf_gated_linear_plan(P(x), P(W), I64(M), I64(F), I64(K), code, buf, 96) == 0
    return buf.value.decode()

"""Sizes at which the 4-bit layer takes each kernel variant on 256 CUs, one
weight or one per group of rows, with every width of the scale groups, and
sizes whose scales pass through LDS in several parts.  The CPU tests hold the
lists to the library's own choice, the GPU tests run them."""
from __future__ import annotations

import ctypes
import os

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
I64 = ctypes.c_int64

# (columns, waves): rows, outputs and K for one weight; K is made a multiple of
# the scale group, past a whole number of 128 where the group is narrower
DENSE = {
    (16, 8): (5, 200, 640), (16, 16): (13, 650, 8192), (32, 8): (16, 8200, 256), (32, 4): (31, 8210, 384),
    (64, 4): (70, 9900, 256), (64, 8): (200, 1990, 8192),
}
# and rows, groups, outputs and K for one weight per group
GROUPED = {
    (16, 8): (21, 5, 130, 512), (16, 16): (9, 4, 200, 8192), (32, 8): (16, 8, 1030, 384), (32, 4): (16, 8, 2050, 256),
    (64, 4): (333, 8, 1010, 256), (64, 8): (290, 6, 1411, 8192),
}
# rows, groups (0: one weight), outputs, K, scale group, zero points, parts
PARTS = [
    (200, 0, 1990, 5504, 32, True, 2),      # 64 columns, 172 scale rows where 168 fit
    (380, 0, 1100, 11008, 32, True, 3),     # 344
    (100, 0, 3650, 8256, 32, False, 2),     # 258 where 256 fit
    (380, 0, 1100, 11008, 64, True, 2),     # 172 of 64
    (70, 0, 9900, 5376, 32, True, 1),       # 168: just one part
    (20, 0, 8200, 10912, 32, True, 2),      # 32 columns, 341 where 340 fit
    (16, 0, 8200, 16448, 32, False, 2),     # 514 where 512 fit
    (3, 0, 70, 32800, 32, False, 2),        # 16 columns, 1025 where 1024 fit
    (17, 0, 50, 43648, 64, True, 2),        # 682 where 680 fit
    (70, 0, 10000, 21632, 128, True, 2),    # 169 of 128
    (90, 0, 8300, 43264, 256, True, 2),     # 169 of 256
    (16, 8, 2050, 10912, 32, True, 2),      # per group of rows
    (290, 6, 1411, 11008, 32, True, 3),
    (290, 6, 1411, 11008, 64, True, 2),
    (9, 4, 70, 32832, 32, False, 2),
]


def variant_cases():
    """(rows, groups or 0, N, K, scale group, zeros, columns, waves)."""
    out = []
    for G in (32, 64, 128, 256):
        for zeros in (False, True):
            for (cols, waves), (R, N, K) in DENSE.items():
                out.append((R, 0, N, K + (G if G < 128 else 0), G, zeros, cols, waves))
            for (cols, waves), (R, E, N, K) in GROUPED.items():
                out.append((R, E, N, K + (G if G < 128 else 0), G, zeros, cols, waves))
    return [c for c in out if c[3] % c[4] == 0]


def plan(R, E, N, K, G, zeros):
    so = ctypes.CDLL(os.path.join(ROOT, "scaffolding_amd", "libsfgemm.so"))
    buf = ctypes.create_string_buffer(96)
    assert so.sf_linear_q4_plan(I64(R), I64(max(1, E)), I64(N), I64(K), I64(G), int(zeros), int(E > 0), buf, 96) == 0
    return buf.value.decode()

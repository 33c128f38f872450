"""Run by tests/test_q4_gpu.py in a child process: takes the device's memory
but for a rest smaller than a 4-bit layer's weight in 16 bits, then runs that
layer on many rows.  Prints one JSON line."""
from __future__ import annotations

import ctypes
import json
import os
import sys

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
for p in (ROOT, HERE):
    if p not in sys.path:
        sys.path.insert(0, p)

from helpers import cu, down, gemm_bound, rnd, up  # noqa: E402
from oracle import experts as ox  # noqa: E402

P, SZ = ctypes.c_void_p, ctypes.c_size_t
MB = 1 << 20


def main() -> None:
    g = cu()
    lib = ctypes.CDLL(os.path.join(ROOT, "scaffolding_amd", "libsfgemm.so"))
    g.set_device(0)
    M, N, K, G = 400, 8192, 16384, 128  # 64 MB packed, 256 MB in 16 bits
    rng = np.random.default_rng(8)
    x = rnd(rng, (M, K), 1.0, "bfloat16")
    q, s = rng.integers(0, 256, (N, K // 2), dtype=np.uint8), np.abs(rnd(rng, (K // G, N), 0.01, "bfloat16"))
    xt, qt, st = up(x, "bfloat16"), g.gputensor_from_numpy(q), up(s, "bfloat16")
    few = up(x[:5], "bfloat16")
    want_few = down(g.dev_linear_q4(few, qt, st))  # code loaded, queue made
    room = g.empty((M, N), g.BFLOAT16)
    g.device_synchronize()
    held = []
    size = 64 * 1024 * MB
    while size >= 32 * MB:
        ptr = P()
        if lib.sf_malloc(ctypes.byref(ptr), SZ(size)) == 0:
            held.append(ptr)
        else:
            size //= 2
    del room  # the result's own memory goes back to the pool
    error = ""
    try:
        y = g.dev_linear_q4(xt, qt, st)
        again = down(g.dev_linear_q4(few, qt, st))
        y = down(y)
    except RuntimeError as e:
        error = str(e)
    for ptr in held:
        lib.sf_free(ptr)
    worst, same = -1.0, False
    if not error:
        same = bool(np.array_equal(again, want_few))
        rows, cols = np.array([0, 15, 16, 383, M - 1]), rng.choice(N, 64, replace=False)
        w = ox.q4_weight(q[cols], s[:, cols])
        y64 = x[rows].astype(np.float64) @ w.T
        # terms of up to 31 |x| s each (16 + q, and the offset taken out again)
        mag = 31.0 * np.abs(x[rows]).astype(np.float64) @ np.repeat(s[:, cols].T.astype(np.float64), G, -1).T
        # unrounded weights: half an ulp of the result and the fp32 sums
        worst = float(np.max(np.abs(y[np.ix_(rows, cols)] - y64) / gemm_bound(y64, mag, 2 * K, "bfloat16")))
    print(json.dumps({"error": error, "held": len(held), "same": same, "worst": worst}), flush=True)


if __name__ == "__main__":
    main()

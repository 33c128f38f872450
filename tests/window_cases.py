"""Windowed attention at sizes that fill the chip, with what they launch on 256
CUs, and its rows in 64 bits over whole arrays; shared by the host's and the
GPU's tests."""
from __future__ import annotations

import ctypes
import os

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
I64 = ctypes.c_int64

# dtype, B, N, H, Hk, D, window, sinks, lengths, launches
LARGE = [
    ("bfloat16", 4, 321, 16, 4, 128, None, 0, None, "window 128 rows, heads up to 128"),
    ("float16", 3, 500, 24, 8, 128, 130, 3, [500, 77, 384], "window 128 rows, heads up to 128"),
    ("float16", 4, 321, 16, 4, 72, 100, 5, [321, 0, 200, 129], "window 128 rows, heads up to 96"),
    ("bfloat16", 2, 1025, 8, 1, 96, 300, 70, None, "window 128 rows, heads up to 96"),
    ("bfloat16", 8, 321, 16, 4, 64, 64, 65, None, "window 128 rows, heads up to 64"),
    ("float16", 9, 257, 16, 16, 40, None, 0, [257, 1, 128, 130, 0, 256, 5, 200, 255], "window 128 rows, heads up to 64"),
]

# dtype, B, n, H, Hk, D, S, window, sinks, launches
CACHED = [
    ("bfloat16", 2, 257, 32, 4, 128, 1500, None, 0, "window 128 rows, heads up to 128"),
    ("float16", 4, 200, 40, 8, 64, 500, 90, 3, "window 128 rows, heads up to 64"),
    ("bfloat16", 6, 150, 24, 8, 80, 400, 90, 10, "window 128 rows, heads up to 96"),
    ("float16", 1, 1, 8, 2, 96, 3000, None, 0, "window split 8, heads up to 96"),
    ("bfloat16", 2, 1, 8, 2, 88, 2000, 1000, 3, "window split 3, heads up to 96"),
    ("bfloat16", 1, 1, 8, 2, 64, 3000, 1500, 0, "window split 6, heads up to 64"),
    ("float16", 1, 2, 8, 2, 128, 3000, 1500, 4, "window split 5, heads up to 128"),
    ("bfloat16", 5, 1, 4, 4, 64, 300, 64, 4, "window split 1, heads up to 64"),
    ("float16", 2, 3, 6, 2, 72, 333, 50, 33, "window split 1, heads up to 96"),
    ("bfloat16", 16, 1, 40, 8, 128, 260, 128, 4, "window split 1, heads up to 128"),
]


def plan(B, H, Hk, rows, capacity, D, window, sinks):
    so = ctypes.CDLL(os.path.join(ROOT, "scaffolding_amd", "libsfgemm.so"))
    buf = ctypes.create_string_buffer(96)
    assert so.sf_window_attention_plan(*map(I64, (B, H, Hk, rows, capacity, D, window or 0, sinks)), buf, 96) == 0
    return buf.value.decode()


def rows64(q, k, v, first, window, sinks, scale):
    """One head's queries at positions first, first + 1, ... over the keys 0, 1,
    ...: (output, log-sums, weights, sum of p |v|, largest sum |q| |k| of a seen
    key); a row without a key gives 0 and -inf."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    i, j = first + np.arange(len(q))[:, None], np.arange(len(k))[None]
    sees = (j <= i) & (((j > i - window) if window is not None else True) | (j < sinks))
    s = np.where(sees, scale * (q @ k.T), -np.inf)
    m = s.max(1, initial=-np.inf, keepdims=True)
    e = np.where(sees, np.exp(s - np.where(np.isinf(m), 0.0, m)), 0.0)
    total = e.sum(1, keepdims=True)
    p = e / np.where(total == 0, 1.0, total)
    with np.errstate(divide="ignore"):
        lse = (m + np.log(total))[:, 0]
    size = np.where(sees, np.abs(q) @ np.abs(k).T, 0.0).max(1, initial=0.0)
    return p @ v, lse, p, p @ np.abs(v), size

"""Gated feed-forward projections and their gradients on the GPU against the
fp64 oracle."""
from __future__ import annotations

import numpy as np
import pytest

from helpers import check_bound, cu, down, out_half_ulp_rel, rnd, up
from oracle import block as ob

pytestmark = pytest.mark.gpu


def bounds(pre, mag, K, dtype, act):
    """Of y and pre: K fp32 sums either projection (2^-23 a term), the slope of
    either activation at most 1.13, a few steps of the activation, and one
    rounding."""
    F = pre.shape[1] // 2
    acc = (K + 4) * 2.0 ** -23 * mag
    hu = out_half_ulp_rel(dtype)
    a = np.abs(ob.gate_act(pre[:, :F], act))
    eg, eu, u = 1.2 * acc[:, :F] + 4e-6 * a, acc[:, F:], np.abs(pre[:, F:])
    y = a * u
    sub = 2.0 ** -25 if dtype == "float16" else 1e-30
    return eg * (u + eu) + a * eu + hu * (y + eg * (u + eu) + a * eu) + sub + 1e-9, acc + hu * np.abs(pre) + sub


CASES = [
    # dtype, M, K, F: every kernel of the table
    ("bfloat16", 1, 4096, 352), ("float16", 16, 520, 77), ("bfloat16", 7, 8, 1), ("float16", 3, 64, 33),  # skinny
    ("bfloat16", 20, 256, 96), ("float16", 33, 72, 17),          # 32 x 64
    ("bfloat16", 300, 320, 500), ("float16", 129, 64, 65),       # 64 x 64
    ("bfloat16", 700, 1000, 1500),                               # 128 x 128
    ("bfloat16", 700, 256, 3000), ("float16", 1029, 384, 1283),  # 256 x 256
    ("bfloat16", 2100, 128, 2305), ("float16", 4200, 128, 2050),  # more tiles than CUs: one workgroup a CU
    ("float16", 5, 1001, 130), ("bfloat16", 333, 1001, 1283), ("float16", 40, 37, 9), ("bfloat16", 1, 1, 1),  # unaligned
    ("bfloat16", 900, 2001, 1400),
    ("float32", 1, 64, 30), ("float32", 70, 129, 77), ("float32", 512, 512, 512),
]


@pytest.mark.parametrize("dtype,M,K,F", CASES)
@pytest.mark.parametrize("act,bias", [("silu", False), ("gelu", True), (None, True)])
def test_forward(dtype, M, K, F, act, bias):
    rng = np.random.default_rng(M + K + F)
    x, W = rnd(rng, (M, K), 1.0, dtype), rnd(rng, (2 * F, K), K ** -0.5, dtype)
    b = rnd(rng, (2 * F,), 0.5, dtype) if bias else None
    gx, gW, gb = up(x, dtype), up(W, dtype), up(b, dtype) if bias else None
    want, pre, mag = ob.gated(x, W, b, act)
    ty, tp = bounds(pre, mag, K, dtype, act)
    y = down(cu().dev_gated_linear(gx, gW, gb, act))
    check_bound(y, want, ty, "y")
    y2, p = cu().dev_gated_linear(gx, gW, gb, act, True)
    assert (down(y2) == y).all()  # the same whether pre is kept or not
    check_bound(down(p), pre, tp, "pre")


@pytest.mark.parametrize("dtype,M,K,F", [
    ("bfloat16", 1, 64, 32), ("float16", 33, 72, 17), ("bfloat16", 257, 130, 100), ("float16", 300, 256, 200),
    ("float32", 33, 50, 41), ("bfloat16", 5, 1, 1),
])
@pytest.mark.parametrize("act,bias", [("silu", True), ("gelu", False), (None, True)])
def test_backward(dtype, M, K, F, act, bias):
    rng = np.random.default_rng(M + K + F)
    x, W = rnd(rng, (M, K), 1.0, dtype), rnd(rng, (2 * F, K), K ** -0.5, dtype)
    g, pre = rnd(rng, (M, F), 0.5, dtype), rnd(rng, (M, 2 * F), 1.5, dtype)
    dx, dw, db = cu().dev_gated_linear_backward(up(g, dtype), up(x, dtype), up(W, dtype), up(pre, dtype), bias, act)
    wx, ww, wb, d = ob.gated_backward(g, x, W, pre, act)
    hu = out_half_ulp_rel(dtype)
    # d is rounded once ahead of the products (its own fp32 error: a few steps
    # of terms whose slopes cancel to less than their size, 1.2 |g up|)
    gate, u = np.abs(pre[:, :F]), np.abs(pre[:, F:])
    size = np.concatenate([np.abs(g) * u * 1.2, np.abs(g) * (gate + 1e-3)], 1)
    sub = 2.0 ** -25 if dtype == "float16" else 0.0
    ed = 8e-6 * size + hu * np.abs(d) + sub
    ad = np.abs(d) + ed
    check_bound(down(dx), wx, ed @ np.abs(W) + 2 * F * 2.0 ** -23 * (ad @ np.abs(W)) + hu * (np.abs(wx) + ed @ np.abs(W)) + sub + 1e-9, "dx")
    check_bound(down(dw), ww, ed.T @ np.abs(x) + M * 2.0 ** -23 * (ad.T @ np.abs(x)) + hu * (np.abs(ww) + ed.T @ np.abs(x)) + sub + 1e-9, "dw")
    assert (db is None) == (not bias)
    if bias:
        check_bound(down(db), wb, ed.sum(0) + M * 2.0 ** -23 * ad.sum(0) + hu * (np.abs(wb) + ed.sum(0)) + sub + 1e-9, "db")


def test_leading_axes_and_empty():
    g = cu()
    rng = np.random.default_rng(0)
    x, W = rnd(rng, (2, 3, 64), 1.0, "bfloat16"), rnd(rng, (20, 64), 0.1, "bfloat16")
    y, p = g.dev_gated_linear(up(x, "bfloat16"), up(W, "bfloat16"), None, "silu", True)
    assert tuple(y.shape) == (2, 3, 10) and tuple(p.shape) == (2, 3, 20)
    flat = g.dev_gated_linear(up(x.reshape(6, 64), "bfloat16"), up(W, "bfloat16"))
    assert (down(flat).reshape(2, 3, 10) == down(y)).all()
    for dtype in ("float32", "bfloat16"):
        e = g.empty((0, 64), g.resolve_dtype(dtype))
        assert tuple(g.dev_gated_linear(e, up(W, dtype)).shape) == (0, 10)
        k0 = g.dev_gated_linear(g.empty((3, 0), g.resolve_dtype(dtype)), g.empty((4, 0), g.resolve_dtype(dtype)),
                                up(np.array([1.0, 2.0, 3.0, 4.0], np.float32), dtype), None)
        assert down(k0).tolist() == [[3.0, 8.0]] * 3  # no terms: the biases' product
    dx, dw, db = g.dev_gated_linear_backward(g.empty((0, 10)), g.empty((0, 64)), up(W, "float32"), g.empty((0, 20)),
                                             True)
    assert (down(dw) == 0).all() and (down(db) == 0).all()


@pytest.mark.parametrize("M,K,F", [(4, 128, 40), (300, 256, 520), (40, 37, 33)])
def test_operands_at_any_element(M, K, F):
    """Operands one element past an aligned address, through the C entry."""
    import ctypes
    import os

    g = cu()
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    lib = ctypes.CDLL(os.path.join(root, "scaffolding_amd", "libsfgemm.so"))
    I64, P = ctypes.c_int64, ctypes.c_void_p
    rng = np.random.default_rng(3)
    x, W, b = rnd(rng, (M, K), 1.0, "bfloat16"), rnd(rng, (2 * F, K), K ** -0.5, "bfloat16"), rnd(rng, (2 * F,), 0.5, "bfloat16")
    want, pre, mag = ob.gated(x, W, b, "silu")
    ty, tp = bounds(pre, mag, K, "bfloat16", "silu")
    for odd in range(5):
        def put(a, i):
            flat = np.concatenate([np.zeros(1 if i == odd else 0, np.float32), a.reshape(-1)])
            return up(flat, "bfloat16"), 2 * (i == odd)
        (gx, ox), (gw, ow), (gb, obb) = put(x, 0), put(W, 1), put(b, 2)
        y, p = g.zeros((M * F + 2,), g.BFLOAT16), g.zeros((2 * M * F + 2,), g.BFLOAT16)
        oy, op = 2 * (odd == 3), 2 * (odd == 4)
        assert lib.sf_gated_linear(P(gx.data_ptr + ox), P(gw.data_ptr + ow), P(gb.data_ptr + obb), P(y.data_ptr + oy),
                                   P(p.data_ptr + op), I64(M), I64(F), I64(K), 2, 4, None) == 0
        y, p = down(y), down(p)
        check_bound(y[oy // 2:][:M * F].reshape(M, F), want, ty, "y %d" % odd)
        check_bound(p[op // 2:][:2 * M * F].reshape(M, 2 * F), pre, tp, "pre %d" % odd)
        assert (y[oy // 2 + M * F:] == 0).all() and (p[op // 2 + 2 * M * F:] == 0).all()

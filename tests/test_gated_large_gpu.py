"""Gated layers on the 256 x 256 tiles (plain, one workgroup a CU walking
several, part rounds as quarters in a second launch) against fp64: every output
of both projections and of their product."""
from __future__ import annotations

import ctypes
import os

import numpy as np
import pytest

from gated_cases import LARGE, plan
from helpers import check_bound, cu, down, out_half_ulp_rel, rnd, up
from oracle import block as ob

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def make(dtype, M, K, F, bias):
    rng = np.random.default_rng(M + F)
    x, W = rnd(rng, (M, K), 1.0, dtype), rnd(rng, (2 * F, K), K ** -0.5, dtype)
    return x, W, rnd(rng, (2 * F,), 0.5, dtype) if bias else None


def expect(x, W, b, dtype, act):
    """(y, bound, pre, bound): K fp32 sums either projection, 2^-23 a term, over
    terms of sizes up to |x| |w| (norms, at least the sum of sizes); the slope of
    either activation at most 1.13 and a few steps of it; one rounding."""
    x, W = x.astype(np.float64), W.astype(np.float64)
    K, F = x.shape[1], len(W) // 2
    pre = x @ W.T
    mag = np.outer(np.sqrt((x * x).sum(1)), np.sqrt((W * W).sum(1)))
    if b is not None:
        pre += b
        mag += np.abs(b)
    acc = (K + 4) * 2.0 ** -23 * mag
    hu, sub = out_half_ulp_rel(dtype), 2.0 ** -25 if dtype == "float16" else 1e-30
    a = ob.gate_act(pre[:, :F], act)
    y, a, u = a * pre[:, F:], np.abs(a), np.abs(pre[:, F:])
    eg, eu = 1.2 * acc[:, :F] + 4e-6 * a, acc[:, F:]
    ey = eg * (u + eu) + a * eu
    return y, ey + hu * (np.abs(y) + ey) + sub + 1e-9, pre, acc + hu * (np.abs(pre) + acc) + sub


@pytest.mark.parametrize("dtype,M,K,F,launches", LARGE)
@pytest.mark.parametrize("act,bias", [("silu", False), ("gelu", True)])
def test_large_tiles(dtype, M, K, F, launches, act, bias):
    x, W, b = make(dtype, M, K, F, bias)
    gx, gW, gb = up(x, dtype), up(W, dtype), up(b, dtype) if bias else None
    assert plan(dtype, M, K, F, gx.data_ptr, gW.data_ptr) == launches
    y, pre = cu().dev_gated_linear(gx, gW, gb, act, True)
    wy, ty, wp, tp = expect(x, W, b, dtype, act)
    check_bound(down(pre), wp, tp, "pre")
    check_bound(down(y), wy, ty, "y")
    assert (down(cu().dev_gated_linear(gx, gW, gb, act)) == down(y)).all()  # the same whether pre is kept or not


@pytest.mark.parametrize("dtype,M,K,F,launches", [LARGE[4], LARGE[5]])
def test_large_tiles_write_their_rows_only(dtype, M, K, F, launches):
    """Results one element past an aligned address, in larger memory: nothing is
    written ahead of them or behind them."""
    x, W, b = make(dtype, M, K, F, True)
    gx, gW, gb = up(x, dtype), up(W, dtype), up(b, dtype)
    want, pre = cu().dev_gated_linear(gx, gW, gb, "silu", True)
    want, pre = down(want).reshape(-1), down(pre).reshape(-1)
    lib, I64, P = ctypes.CDLL(os.path.join(ROOT, "scaffolding_amd", "libsfgemm.so")), ctypes.c_int64, ctypes.c_void_p
    Y, p = (cu().zeros((n + 65,), gx.dtype) for n in (M * F, 2 * M * F))
    code = {"float16": 1, "bfloat16": 2}[dtype]
    assert lib.sf_gated_linear(P(gx.data_ptr), P(gW.data_ptr), P(gb.data_ptr), P(Y.data_ptr + 2), P(p.data_ptr + 2), I64(M),
                               I64(F), I64(K), code, 4, None) == 0
    for got, w in ((down(Y), want), (down(p), pre)):
        assert np.array_equal(got[1:len(w) + 1], w) and got[0] == 0 and not got[len(w) + 1:].any()


def test_quarters_captured_and_replayed():
    """Both launches in a graph: every replay gives the eager result, with eager
    calls between."""
    dtype, M, K, F, launches = LARGE[5]
    x, W, _ = make(dtype, M, K, F, False)
    g = cu()
    gx, gW = up(x, dtype), up(W, dtype)
    other = up(-x, dtype)
    want = down(g.dev_gated_linear(gx, gW))
    y, lib, hip = g.zeros((M, F), gx.dtype), ctypes.CDLL(os.path.join(ROOT, "scaffolding_amd", "libsfgemm.so")), ctypes.CDLL(
        "libamdhip64.so.7")
    I64, P = ctypes.c_int64, ctypes.c_void_p
    st, graph, ex = P(), P(), P()
    assert lib.sf_stream_create(ctypes.byref(st)) == 0
    g.device_synchronize()
    assert hip.hipStreamBeginCapture(st, 0) == 0
    rc = lib.sf_gated_linear(P(gx.data_ptr), P(gW.data_ptr), None, P(y.data_ptr), None, I64(M), I64(F), I64(K), 2, 4, st)
    assert hip.hipStreamEndCapture(st, ctypes.byref(graph)) == 0 and rc == 0
    assert hip.hipGraphInstantiate(ctypes.byref(ex), graph, None, None, ctypes.c_size_t(0)) == 0
    for _ in range(3):
        g.dev_gated_linear(other, gW)
        g.device_synchronize()
        assert lib.sf_zero(P(y.data_ptr), ctypes.c_size_t(y.nbytes), st) == 0
        assert hip.hipGraphLaunch(ex, st) == 0 and lib.sf_stream_synchronize(st) == 0
        assert np.array_equal(down(y), want)
    hip.hipGraphExecDestroy(ex)
    hip.hipGraphDestroy(graph)
    lib.sf_stream_destroy(st)

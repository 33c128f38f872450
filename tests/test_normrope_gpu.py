"""Norms of queries and keys with the rotation, on the GPU against the fp64
oracle."""
from __future__ import annotations

import numpy as np
import pytest

from helpers import check_bound, cu, down, out_half_ulp_rel, quantize, rnd, up
from oracle import block as ob

pytestmark = pytest.mark.gpu


def ints(a):
    return cu().gputensor_from_numpy(np.ascontiguousarray(a, np.int32))


def f32(a):
    return cu().gputensor_from_numpy(np.ascontiguousarray(a, np.float32))


def make(rng, dtype, B, N, H, Hk, D, R, P, affine=True, layer=False):
    x = rnd(rng, (B, N, (H + 2 * Hk) * D), 1.0, dtype)
    table = ob.rope_table(P, R).astype(np.float32) if R else None
    w = quantize((rng.random((2, D)) + 0.5).astype(np.float32), dtype) if affine else None
    b = rnd(rng, (2, D), 0.3, dtype) if affine and layer else None
    return x, table, w, b


def dev(t, dtype):
    return None if t is None else up(t, dtype)


def steps(D):
    """fp32 roundings between x and a normed, turned column: the sum of D
    squares (at most D of them, half of it in 1 / sqrt), the mean's D, and a
    few for the products."""
    return (2 * D + 16) * 2.0 ** -24


CASES = [
    # dtype, B, N, H, Hk, D, R, norm, interleaved
    ("bfloat16", 1, 1, 1, 1, 128, 128, "rms", False),
    ("bfloat16", 2, 5, 4, 2, 128, 128, "rms", True),
    ("float16", 3, 7, 5, 1, 64, 32, "layer", False),
    ("bfloat16", 1, 333, 3, 3, 64, 64, "layer", True),
    ("float32", 2, 9, 2, 1, 128, 128, "layer", False),
    ("float32", 1, 70, 8, 8, 32, 32, "rms", True),
    ("float16", 1, 11, 3, 1, 72, 72, "rms", False),     # halves of 36: chunks of 4
    ("bfloat16", 2, 6, 2, 2, 96, 48, "rms", False),
    ("float16", 1, 5, 2, 1, 256, 256, "layer", False),
    ("bfloat16", 1, 4, 2, 1, 256, 24, "rms", True),     # most of the head unturned
    ("float32", 1, 4, 2, 1, 255, 254, "rms", False),    # single columns, two pairs a lane
    ("float16", 2, 3, 3, 2, 37, 10, "layer", True),
    ("bfloat16", 1, 3, 2, 1, 7, 6, "layer", False),
    ("float32", 1, 3, 1, 1, 1, 0, "rms", False),
    ("bfloat16", 2, 4, 2, 1, 40, 0, "rms", False),      # no rotation
    ("bfloat16", 1, 5000, 1, 1, 64, 64, "rms", False),  # several tokens a wave
]


@pytest.mark.parametrize("dtype,B,N,H,Hk,D,R,norm,inter", CASES)
@pytest.mark.parametrize("affine", [True, False])
def test_forward(dtype, B, N, H, Hk, D, R, norm, inter, affine):
    rng = np.random.default_rng(N + D)
    x, table, w, b = make(rng, dtype, B, N, H, Hk, D, R, N + 3, affine, norm == "layer")
    pos = rng.integers(0, N + 3, (B, N)) if affine else np.tile(np.arange(N), (B, 1))
    y = down(cu().dev_qk_norm_rope(up(x, dtype), H, Hk, None if table is None else f32(table), dev(w, dtype),
                                   dev(b, dtype), norm, 1e-6, ints(pos) if affine else None, inter))
    want, mag = ob.qk_norm_rope(x, H, Hk, table, pos, w, b, norm, 1e-6, inter)
    hu = out_half_ulp_rel(dtype)
    check_bound(y, want, steps(D) * mag + hu * np.abs(want) + 1e-7)
    v = (H + Hk) * D
    assert (y[..., v:] == x[..., v:]).all()  # values go through


@pytest.mark.parametrize("dtype,B,N,H,Hk,D,R,norm,inter", CASES)
@pytest.mark.parametrize("affine", [True, False])
def test_backward(dtype, B, N, H, Hk, D, R, norm, inter, affine):
    rng = np.random.default_rng(N + D + 1)
    x, table, w, _ = make(rng, dtype, B, N, H, Hk, D, R, N + 3, affine)
    g = rnd(rng, x.shape, 0.5, dtype)
    pos = rng.integers(0, N + 3, (B, N)) if affine else np.tile(np.arange(N), (B, 1))
    tab = None if table is None else f32(table)
    args = (up(g, dtype), up(x, dtype), H, Hk, tab, dev(w, dtype), norm, 1e-6, ints(pos) if affine else None, inter)
    dx, dw, db = cu().dev_qk_norm_rope_backward(*args)
    (wx, ww, wb), (mx, mw, mb) = ob.qk_norm_rope_backward(g, x, H, Hk, table, pos, w, norm, 1e-6, inter)
    hu = out_half_ulp_rel(dtype)
    check_bound(down(dx), wx, 3 * steps(D) * mx + hu * np.abs(wx) + 1e-7, "dx")
    n = B * N * max(H, Hk)  # terms of the longest sum
    check_bound(down(dw), ww, (steps(D) + n * 2.0 ** -24) * mw + hu * np.abs(ww) + 1e-7, "dw")
    assert (db is None) == (norm == "rms")
    if db is not None:
        check_bound(down(db), wb, (n + 4) * 2.0 ** -24 * mb + hu * np.abs(wb) + 1e-7, "db")
    again = cu().dev_qk_norm_rope_backward(*args)
    for a, c in zip((dx, dw, db), again):
        assert a is None or (down(a) == down(c)).all()


@pytest.mark.parametrize("dtype,B,n,H,Hk,D,R,S,norm", [
    ("bfloat16", 3, 1, 4, 2, 128, 128, 20, "rms"), ("float16", 4, 5, 3, 1, 72, 36, 17, "layer"),
    ("float32", 2, 3, 2, 2, 33, 32, 9, "rms"), ("bfloat16", 1, 130, 8, 8, 64, 64, 200, "rms"),
])
def test_cached(dtype, B, n, H, Hk, D, R, S, norm):
    """New rows go behind the lengths; every other row of the caches, and those
    past the capacity, stay out of it."""
    rng = np.random.default_rng(n)
    x, table, w, b = make(rng, dtype, B, n, H, Hk, D, R, S + n, True, norm == "layer")
    k, v = rnd(rng, (B, S, Hk * D), 1.0, dtype), rnd(rng, (B, S, Hk * D), 1.0, dtype)
    lengths = rng.integers(0, S - n + 1, B)
    lengths[0] = S - n
    if B > 1:
        lengths[1] = S - 1  # the last of its new rows is past the capacity (n > 1)
    gk, gv = up(k, dtype), up(v, dtype)
    q = down(cu().dev_qk_norm_rope_cached(up(x, dtype), H, Hk, f32(table), gk, gv, ints(lengths), dev(w, dtype),
                                          dev(b, dtype), norm))
    pos = lengths[:, None] + np.arange(n)
    y, mag = ob.qk_norm_rope(x, H, Hk, table, pos, w, b, norm)
    tol = steps(D) * mag + out_half_ulp_rel(dtype) * np.abs(y) + 1e-7
    check_bound(q, y[..., :H * D], tol[..., :H * D], "q")
    wk, wv, tk = k.astype(np.float64), v.copy(), np.zeros(k.shape)
    for s in range(B):
        m = min(n, S - lengths[s])
        wk[s, lengths[s]:lengths[s] + m] = y[s, :m, H * D:(H + Hk) * D]
        tk[s, lengths[s]:lengths[s] + m] = tol[s, :m, H * D:(H + Hk) * D]
        wv[s, lengths[s]:lengths[s] + m] = x[s, :m, (H + Hk) * D:]
    check_bound(down(gk), wk, tk, "k")
    assert (down(gv) == wv).all()


def test_positions_that_the_table_lacks_give_nan():
    rng = np.random.default_rng(0)
    x, table, w, _ = make(rng, "bfloat16", 1, 6, 2, 1, 64, 32, 4)
    pos = np.array([[0, 3, 4, -1, 2 ** 31 - 1, -2 ** 31]])
    y = down(cu().dev_qk_norm_rope(up(x, "bfloat16"), 2, 1, f32(table), up(w, "bfloat16"), None, "rms", 1e-6, ints(pos)))
    h = y.reshape(6, 4, 64)
    assert np.isfinite(h[:2]).all() and np.isnan(h[2:, :3, :32]).all()
    assert np.isfinite(h[2:, :3, 32:]).all() and np.isfinite(h[:, 3]).all()


def test_lengths_out_of_range_write_nothing():
    rng = np.random.default_rng(0)
    x, table, w, _ = make(rng, "bfloat16", 4, 2, 2, 1, 64, 64, 8)
    k = rnd(rng, (4, 5, 64), 1.0, "bfloat16")
    gk, gv = up(k, "bfloat16"), up(k, "bfloat16")
    cu().dev_qk_norm_rope_cached(up(x, "bfloat16"), 2, 1, f32(table), gk, gv, ints([-2, 5, 2 ** 31 - 1, -2 ** 31]),
                                 up(w, "bfloat16"))
    assert (down(gk) == k).all() and (down(gv) == k).all()


def test_a_head_of_zeros_and_non_finite_heads():
    """0 r = 0 with r = 1 / sqrt(eps); a NaN or infinite head spoils itself
    alone."""
    rng = np.random.default_rng(0)
    for dtype in ("float32", "bfloat16"):
        x, table, w, _ = make(rng, dtype, 1, 4, 2, 1, 64, 64, 4)
        x[0, 0, :64] = 0.0
        x[0, 1, 64 + 5] = np.nan
        x[0, 2, 128 + 9] = np.inf
        y = down(cu().dev_qk_norm_rope(up(x, dtype), 2, 1, f32(table), up(w, dtype))).reshape(4, 4, 64)
        assert (y[0, 0] == 0).all() and np.isnan(y[1, 1]).all() and np.isnan(y[2, 2]).any()
        fine = np.isfinite(y).all(-1)
        assert fine.sum() == 14 and not fine[1, 1] and not fine[2, 2]


def test_empty():
    g = cu()
    x = g.empty((2, 0, 4 * 64), np.float32)
    assert tuple(g.dev_qk_norm_rope(x, 2, 1).shape) == (2, 0, 256)
    dx, dw, db = g.dev_qk_norm_rope_backward(x, x, 2, 1, None, None, "layer")
    assert tuple(dx.shape) == (2, 0, 256) and (down(dw) == 0).all() and (down(db) == 0).all()


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("dtype,D,H,Hk", [
    ("bfloat16", 64, 5, 1), ("float16", 64, 8, 3), ("bfloat16", 128, 30, 3), ("float32", 128, 4, 1),
    ("float16", 256, 3, 1), ("float32", 37, 3, 2),
])
def test_backward_without_eps(dtype, D, H, Hk, norm):
    """eps 0 with heads that leave lanes of a wave over: those lanes hold no head
    and add nothing to the parameters' gradients."""
    rng = np.random.default_rng(D + H)
    B, N, R = 2, 9, D // 2 * 2
    x, table, w, _ = make(rng, dtype, B, N, H, Hk, D, R, N)
    g = rnd(rng, x.shape, 0.5, dtype)
    pos = np.tile(np.arange(N), (B, 1))
    dx, dw, db = cu().dev_qk_norm_rope_backward(up(g, dtype), up(x, dtype), H, Hk, f32(table), up(w, dtype), norm, 0.0)
    (wx, ww, wb), (mx, mw, mb) = ob.qk_norm_rope_backward(g, x, H, Hk, table, pos, w, norm, 0.0)
    hu = out_half_ulp_rel(dtype)
    n = B * N * max(H, Hk)
    check_bound(down(dx), wx, 3 * steps(D) * mx + hu * np.abs(wx) + 1e-7, "dx")
    assert np.isfinite(down(dw)).all()
    check_bound(down(dw), ww, (steps(D) + n * 2.0 ** -24) * mw + hu * np.abs(ww) + 1e-7, "dw")
    if norm == "layer":
        check_bound(down(db), wb, (n + 4) * 2.0 ** -24 * mb + hu * np.abs(wb) + 1e-7, "db")


@pytest.mark.parametrize("norm,has_bias,given", [("rms", True, True), ("rms", None, False), ("rms", False, False),
                                                 ("layer", True, True), ("layer", None, True), ("layer", False, False)])
def test_gradient_of_a_bias(norm, has_bias, given):
    """Either norm takes a bias and gives its gradient, by formula and by the
    sums' differences: the loss is linear in it, so they are as exact as its own
    fp64."""
    from scaffolding_amd import Tensor
    from scaffolding_amd.nn import functional as F
    rng = np.random.default_rng(5)
    dtype, B, N, H, Hk, D, R = "bfloat16", 2, 7, 3, 2, 64, 32
    x, table, w, _ = make(rng, dtype, B, N, H, Hk, D, R, N)
    g, bias = rnd(rng, x.shape, 0.5, dtype), rnd(rng, (2, D), 0.3, dtype)
    pos = np.tile(np.arange(N), (B, 1))
    t = lambda a, d=dtype: Tensor(a, dtype=d, device="cuda")
    y = F.qk_norm_rope(t(x), H, Hk, t(table, "float32"), t(w), t(bias), norm)
    want, mag = ob.qk_norm_rope(x, H, Hk, table, pos, w, bias, norm)
    hu = out_half_ulp_rel(dtype)
    check_bound(y.numpy(), want, steps(D) * mag + hu * np.abs(want) + 1e-7, "y")
    dx, dw, db = F.qk_norm_rope_backward(t(g), t(x), H, Hk, t(table, "float32"), t(w), norm, has_bias=has_bias)
    (wx, ww, wb), (mx, mw, mb) = ob.qk_norm_rope_backward(g, x, H, Hk, table, pos, w, norm)
    n = B * N * H
    check_bound(dx.numpy(), wx, 3 * steps(D) * mx + hu * np.abs(wx) + 1e-7, "dx")
    check_bound(dw.numpy(), ww, (steps(D) + n * 2.0 ** -24) * mw + hu * np.abs(ww) + 1e-7, "dw")
    assert (db is not None) == given
    if given:
        check_bound(db.numpy(), wb, (n + 4) * 2.0 ** -24 * mb + hu * np.abs(wb) + 1e-7, "db")
        lo, hi = ((ob.qk_norm_rope(x, H, Hk, table, pos, w, bias + s, norm)[0] * g).sum() for s in (-0.5, 0.5))
        assert abs(hi - lo - wb.sum()) < 1e-9 * np.abs(g).sum()

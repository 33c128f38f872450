"""Windowed attention with sinks on the GPU against the fp64 oracle."""
from __future__ import annotations

import numpy as np
import pytest

from helpers import check_bound, cu, down, out_half_ulp_rel, rnd, up
from oracle import block as ob

pytestmark = pytest.mark.gpu


def ints(a):
    return cu().gputensor_from_numpy(np.ascontiguousarray(a, np.int32))


def forward_bound(x, H, Hk, window, sinks, scale, dtype, lengths=None):
    """Per element of the output: the weights are rounded once for their product
    with V (half a step each), scores carry D fp32 roundings (2^-23 a term of
    sum |q k|, times the exponential's slope 1) plus a few steps of the
    exponent, both against sum_j p_j |v_j| twice (the normalisation shares
    them); then one rounding."""
    q, k, v = ob.split_heads(x, H, Hk)
    B, N, _, D = q.shape
    avg = np.zeros((B, N, H, D))
    size = np.zeros((B, N, H, 1))
    for b in range(B):
        n = N if lengths is None else min(max(int(lengths[b]), 0), N)
        for h in range(H):
            u = h // (H // Hk)
            _, _, p = ob.window_rows(q[b, :n, h], k[b, :n, u], v[b, :n, u], 0, window, sinks, scale)
            avg[b, :n, h] = p @ np.abs(v[b, :n, u])
            s = np.abs(q[b, :n, h]) @ np.abs(k[b, :n, u]).T
            size[b, :n, h, 0] = (s * (p > 0)).max(1, initial=0.0)
    hu = out_half_ulp_rel(dtype)
    rel = 2 * hu + 2 * (D * 2.0 ** -23 * abs(scale) * size + 2.0 ** -18)
    return (rel * avg).reshape(B, N, H * D), (D * 2.0 ** -23 * abs(scale) * size[..., 0]).transpose(0, 2, 1)


def check(y, want, tol, dtype, what=""):
    hu = out_half_ulp_rel(dtype)
    check_bound(y, want, tol + hu * (np.abs(want) + tol) + 2.0 ** -24, what)


CASES = [
    # dtype, B, N, H, Hk, D, window, sinks
    ("bfloat16", 1, 1, 1, 1, 128, None, 0), ("float16", 1, 2, 2, 1, 8, 1, 0), ("bfloat16", 2, 63, 2, 2, 64, None, 0),
    ("float16", 1, 64, 4, 1, 40, 64, 0), ("bfloat16", 1, 65, 3, 1, 72, 1, 1), ("float16", 2, 130, 4, 2, 96, 33, 4),
    ("bfloat16", 1, 129, 2, 1, 128, 128, 200), ("float16", 1, 200, 2, 2, 128, 65, 63),
    ("bfloat16", 1, 300, 6, 3, 104, 100, 70), ("float16", 3, 257, 2, 1, 64, 64, 65), ("bfloat16", 1, 500, 8, 8, 64, 37, 3),
    ("float16", 1, 513, 9, 9, 16, 2 ** 40, 0), ("bfloat16", 1, 450, 1, 1, 128, 129, 2 ** 40),
]


@pytest.mark.parametrize("dtype,B,N,H,Hk,D,window,sinks", CASES)
def test_forward(dtype, B, N, H, Hk, D, window, sinks):
    rng = np.random.default_rng(N + D)
    x = rnd(rng, (B, N, (H + 2 * Hk) * D), 1.0, dtype)
    scale = D ** -0.5
    want, lse = ob.window_attention(x, H, Hk, window, sinks, scale)
    tol, tl = forward_bound(x, H, Hk, window, sinks, scale, dtype)
    gx = up(x, dtype)
    check(down(cu().dev_window_attention(gx, H, Hk, window, sinks)), want, tol, dtype)
    y, ls = cu().dev_window_attention(gx, H, Hk, window, sinks, None, None, True)
    check(down(y), want, tol, dtype, "with lse")
    check_bound(down(ls), lse, tl + 2.0 ** -18 + 2.0 ** -22 * np.abs(lse), "lse")


@pytest.mark.parametrize("dtype,N,H,Hk,D,window,sinks,lengths", [
    ("bfloat16", 200, 2, 1, 128, 50, 3, [200, 1, 0, 131, 64, 65]), ("float16", 70, 4, 2, 64, None, 0, [-5, 70, 900, 69]),
    ("bfloat16", 300, 2, 2, 72, 20, 100, [90, 129, 128]),
])
def test_lengths(dtype, N, H, Hk, D, window, sinks, lengths):
    """Keys and rows behind a sequence's end: NaN there changes nothing, and
    those rows give 0."""
    rng = np.random.default_rng(N)
    B = len(lengths)
    x = rnd(rng, (B, N, (H + 2 * Hk) * D), 1.0, dtype)
    for b, n in enumerate(lengths):
        x[b, max(n, 0):] = np.nan
    scale = 0.21
    want, lse = ob.window_attention(x, H, Hk, window, sinks, scale, lengths)
    tol, tl = forward_bound(np.nan_to_num(x), H, Hk, window, sinks, scale, dtype, lengths)
    y, ls = cu().dev_window_attention(up(x, dtype), H, Hk, window, sinks, scale, ints(lengths), True)
    y, ls = down(y), down(ls)
    check(y, want, tol, dtype)
    none = np.isinf(lse)
    assert (np.isneginf(ls) == none).all()
    check_bound(ls[~none], lse[~none], (tl + 2.0 ** -18 + 2.0 ** -22 * np.abs(lse))[~none], "lse")
    for b, n in enumerate(lengths):
        assert (y[b, max(n, 0):] == 0).all()
    plain = down(cu().dev_window_attention(up(x, dtype), H, Hk, window, sinks, scale, ints(lengths)))
    check(plain, want, tol, dtype)


@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0, 40.0])
def test_scales_and_steep_rows(scale):
    """Scores of hundreds, rising and falling along the keys: the references
    move far."""
    rng = np.random.default_rng(1)
    N, H, D = 300, 2, 64
    x = rnd(rng, (1, N, 4 * D), 1.0, "bfloat16")
    x[0, :, 2 * D] = np.linspace(-2, 2, N).astype(np.float32)
    from helpers import quantize
    x = quantize(x, "bfloat16")
    want, lse = ob.window_attention(x, H, 1, 90, 5, scale)
    tol, tl = forward_bound(x, H, 1, 90, 5, scale, "bfloat16")
    y, ls = cu().dev_window_attention(up(x, "bfloat16"), H, 1, 90, 5, scale, None, True)
    check(down(y), want, tol, "bfloat16")
    check_bound(down(ls), lse, tl + 2.0 ** -18 + 2.0 ** -22 * np.abs(lse), "lse")


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_values_that_rows_do_not_see(value):
    """A token whose value row is not finite spoils the rows that see it, and no
    other: not those ahead of it, nor those whose window has left it."""
    rng = np.random.default_rng(2)
    N, H, D, window, sinks = 400, 2, 64, 40, 2
    x = rnd(rng, (1, N, 4 * D), 1.0, "bfloat16")
    at = 150
    x[0, at, 3 * D + 7] = value
    clean = x.copy()
    clean[0, at, 3 * D + 7] = 0.0
    want, _ = ob.window_attention(clean, H, 1, window, sinks, 0.125)
    tol, _ = forward_bound(clean, H, 1, window, sinks, 0.125, "bfloat16")
    y = down(cu().dev_window_attention(up(x, "bfloat16"), H, 1, window, sinks, 0.125)).reshape(N, H, D)
    sees = (np.arange(N) >= at) & (np.arange(N) < at + window)
    assert not np.isfinite(y[sees][:, :, 7]).any()
    y[sees, :, 7] = want.reshape(N, H, D)[sees, :, 7]
    check(y.reshape(1, N, H * D), want, tol, "bfloat16")
    # a key that is not finite makes the scores of the rows that see it NaN
    x = clean.copy()
    x[0, at, 2 * D:3 * D] = np.nan
    y = down(cu().dev_window_attention(up(x, "bfloat16"), H, 1, window, sinks, 0.125)).reshape(N, H, D)
    assert np.isnan(y[sees]).all()
    check(y[~sees].reshape(1, -1, H * D), want.reshape(N, H, D)[~sees].reshape(1, -1, H * D),
          tol.reshape(N, H, D)[~sees].reshape(1, -1, H * D), "bfloat16")


# ---- over a cache ------------------------------------------------------------------

def cached_bound(q, k, v, lengths, H, Hk, window, sinks, scale, dtype):
    B, n, C = q.shape
    D, S = C // H, k.shape[1]
    avg, size = np.zeros((B, n, H, D)), np.zeros((B, n, H, 1))
    for b in range(B):
        keys = min(int(lengths[b]) + n, S)
        for h in range(H):
            u = h // (H // Hk)
            kb, vb = (np.asarray(a, np.float64)[b, :keys].reshape(keys, Hk, D)[:, u] for a in (k, v))
            qb = np.asarray(q, np.float64)[b].reshape(n, H, D)[:, h]
            _, _, p = ob.window_rows(qb, kb, vb, int(lengths[b]), window, sinks, scale)
            avg[b, :, h] = p @ np.abs(vb)
            size[b, :, h, 0] = ((np.abs(qb) @ np.abs(kb).T) * (p > 0)).max(1, initial=0.0)
    hu = out_half_ulp_rel(dtype)
    return ((2 * hu + 2 * (D * 2.0 ** -23 * abs(scale) * size + 2.0 ** -18)) * avg).reshape(B, n, C)


@pytest.mark.parametrize("dtype,B,n,H,Hk,D,S,window,sinks", [
    ("bfloat16", 1, 1, 1, 1, 128, 1, None, 0), ("float16", 3, 1, 8, 2, 128, 700, None, 0),
    ("bfloat16", 5, 1, 4, 4, 64, 300, 64, 4), ("float16", 2, 3, 6, 2, 72, 333, 50, 33), ("bfloat16", 2, 1, 32, 1, 96, 500, 200, 100),
    ("bfloat16", 1, 1, 16, 2, 128, 5000, None, 0), ("float16", 1, 1, 2, 1, 64, 9000, 4000, 5), ("bfloat16", 1, 40, 4, 1, 40, 200, 70, 3),
    ("float16", 2, 150, 4, 2, 128, 400, 90, 10), ("bfloat16", 1, 257, 2, 1, 64, 300, None, 0), ("float16", 1, 5, 3, 1, 8, 64, 1, 0),
    ("bfloat16", 2, 17, 7, 1, 128, 2100, 1000, 1), ("bfloat16", 16, 1, 40, 8, 128, 260, 128, 4),
])
def test_cached(dtype, B, n, H, Hk, D, S, window, sinks):
    """Lengths from none to the whole cache; what lies behind the new tokens is
    NaN."""
    rng = np.random.default_rng(S + n)
    q = rnd(rng, (B, n, H * D), 1.0, dtype)
    k, v = rnd(rng, (B, S, Hk * D), 1.0, dtype), rnd(rng, (B, S, Hk * D), 1.0, dtype)
    lengths = rng.integers(0, S - n + 1, B)
    lengths[0] = S - n
    if B > 1:
        lengths[1] = 0
    for b in range(B):
        k[b, lengths[b] + n:] = np.nan
        v[b, lengths[b] + n:] = np.nan
    scale = D ** -0.5
    want = ob.window_attention_cached(q, k, v, lengths, H, Hk, window, sinks, scale)
    tol = cached_bound(q, k, v, lengths, H, Hk, window, sinks, scale, dtype)
    args = (up(q, dtype), up(k, dtype), up(v, dtype), ints(lengths), H, Hk, window, sinks)
    y = down(cu().dev_window_attention_cached(*args))
    check(y, want, tol, dtype)
    assert (down(cu().dev_window_attention_cached(*args)) == y).all()


def test_cached_lengths_out_of_range():
    """Below 0 counts as 0, past the capacity as the capacity: there a token
    sees what its window reaches of the cache, and 0 comes of nothing."""
    rng = np.random.default_rng(0)
    S, D = 40, 64
    q, k, v = (rnd(rng, (4, m, D), 1.0, "bfloat16") for m in (1, S, S))
    given, cut = [-3, S, 2 ** 31 - 1, S - 1], [0, S, S, S - 1]
    for window in (1, 2, 10):
        want = ob.window_attention_cached(q, k, v, cut, 1, 1, window, 0, 0.125)
        tol = cached_bound(q, k, v, cut, 1, 1, window, 0, 0.125, "bfloat16")
        y = down(cu().dev_window_attention_cached(up(q, "bfloat16"), up(k, "bfloat16"), up(v, "bfloat16"), ints(given),
                                                  1, 1, window, 0, 0.125))
        check(y, want, tol, "bfloat16")
        assert window > 1 or (y[1:3] == 0).all()


@pytest.mark.parametrize("n,S", [(1, 3000), (200, 600)])
def test_cached_values_that_rows_do_not_see(n, S):
    """A NaN among the cache's old values, outside every window."""
    rng = np.random.default_rng(0)
    H, D, window = 4, 64, 100
    q, k, v = rnd(rng, (1, n, H * D), 1.0, "float16"), rnd(rng, (1, S, D), 1.0, "float16"), rnd(rng, (1, S, D), 1.0, "float16")
    length = S - n
    clean = v.copy()
    v[0, length - window] = np.nan  # the last that no new token's window reaches
    want = ob.window_attention_cached(q, k, clean, [length], H, 1, window, 3, 0.125)
    tol = cached_bound(q, k, clean, [length], H, 1, window, 3, 0.125, "float16")
    y = down(cu().dev_window_attention_cached(up(q, "float16"), up(k, "float16"), up(v, "float16"), ints([length]), H, 1,
                                              window, 3, 0.125))
    check(y, want, tol, "float16")


def test_empty():
    g = cu()
    x = g.empty((2, 0, 4 * 64), np.float16)
    y, lse = g.dev_window_attention(x, 2, 1, 4, 1, None, None, True)
    assert tuple(y.shape) == (2, 0, 128) and tuple(lse.shape) == (2, 2, 0)
    q, k = g.empty((2, 0, 128), np.float16), g.empty((2, 5, 64), np.float16)
    assert tuple(g.dev_window_attention_cached(q, k, k, ints([0, 0]), 2, 1).shape) == (2, 0, 128)


# ---- gradients -----------------------------------------------------------------------

def backward_bound(g, x, H, Hk, window, sinks, scale, dtype, lengths=None):
    """Per element of dx, in terms of the sums of magnitudes `mag` that
    ob.window_attention_backward gives (dS by its parts |dP| + |delta|):
      - P and dS are rounded once for their products: half a step each;
      - delta comes of the rounded output (half a step of it) and lse carries
        fp32 errors: both within another half step of the magnitudes;
      - the scores' D fp32 roundings move P by D 2^-23 scale sum |q k|;
      - the sums over up to N rows of every head (or keys) 2^-23 a term.
    fp16's smallest step (2^-24, dS; P is held times 2^8) adds N H of them
    times the operand."""
    want, mag = ob.window_attention_backward(g, x, H, Hk, window, sinks, scale, lengths)
    q, k, v = ob.split_heads(x, H, Hk)
    D, N = q.shape[-1], q.shape[1]
    size = np.abs(q).sum(-1).max() * np.abs(k).max()
    hu = out_half_ulp_rel(dtype)
    rel = 3 * hu + 4 * D * 2.0 ** -23 * abs(scale) * size + (N * H // Hk + D) * 2.0 ** -23 + 2.0 ** -16
    tiny = 2.0 ** -24 * N * (H // Hk) * np.abs(x).max() * max(abs(scale), 1.0) if dtype == "float16" else 0.0
    tol = rel * mag + tiny
    return want, tol + hu * (np.abs(want) + tol) + 2.0 ** -24


BACK = [
    # dtype, B, N, H, Hk, D, window, sinks
    ("bfloat16", 1, 1, 1, 1, 128, None, 0), ("float16", 1, 3, 2, 1, 8, 1, 0), ("bfloat16", 2, 63, 2, 2, 64, None, 0),
    ("float16", 1, 64, 4, 1, 40, 64, 0), ("bfloat16", 1, 65, 3, 1, 72, 1, 1), ("float16", 2, 130, 4, 2, 96, 33, 4),
    ("bfloat16", 1, 129, 2, 1, 128, 128, 200), ("float16", 1, 200, 2, 2, 128, 65, 63),
    ("bfloat16", 1, 300, 6, 3, 104, 100, 70), ("float16", 3, 257, 2, 1, 64, 64, 65), ("bfloat16", 1, 500, 8, 8, 64, 37, 3),
    ("bfloat16", 1, 520, 4, 2, 128, None, 0), ("float16", 1, 700, 2, 1, 128, 50, 150), ("bfloat16", 1, 390, 2, 1, 32, 129, 2 ** 40),
]


@pytest.mark.parametrize("dtype,B,N,H,Hk,D,window,sinks", BACK)
def test_backward(dtype, B, N, H, Hk, D, window, sinks):
    rng = np.random.default_rng(N + D)
    x = rnd(rng, (B, N, (H + 2 * Hk) * D), 1.0, dtype)
    g = rnd(rng, (B, N, H * D), 0.5, dtype)
    gx, gg = up(x, dtype), up(g, dtype)
    out, lse = cu().dev_window_attention(gx, H, Hk, window, sinks, None, None, True)
    dx = down(cu().dev_window_attention_backward(gg, gx, out, lse, H, Hk, window, sinks))
    want, tol = backward_bound(g, x, H, Hk, window, sinks, D ** -0.5, dtype)
    check_bound(dx, want, tol)
    again = down(cu().dev_window_attention_backward(gg, gx, out, lse, H, Hk, window, sinks))
    assert (dx == again).all()


@pytest.mark.parametrize("dtype,N,H,Hk,D,window,sinks,lengths", [
    ("bfloat16", 200, 2, 1, 128, 50, 3, [200, 1, 0, 131, 64, 65]), ("float16", 270, 4, 2, 64, None, 0, [-5, 270, 900, 129]),
    ("bfloat16", 300, 2, 2, 72, 20, 100, [90, 129, 128]),
])
def test_backward_lengths(dtype, N, H, Hk, D, window, sinks, lengths):
    """What lies behind a sequence's end (NaN here) changes nothing, and gets
    0."""
    rng = np.random.default_rng(N)
    B = len(lengths)
    x = rnd(rng, (B, N, (H + 2 * Hk) * D), 1.0, dtype)
    g = rnd(rng, (B, N, H * D), 0.5, dtype)
    clean = x.copy()
    for b, n in enumerate(lengths):
        x[b, max(n, 0):] = np.nan
        g[b, max(n, 0):] = np.nan
    gx, gl = up(x, dtype), ints(lengths)
    out, lse = cu().dev_window_attention(gx, H, Hk, window, sinks, 0.2, gl, True)
    dx = down(cu().dev_window_attention_backward(up(g, dtype), gx, out, lse, H, Hk, window, sinks, 0.2, gl))
    want, tol = backward_bound(np.nan_to_num(g), clean, H, Hk, window, sinks, 0.2, dtype, lengths)
    check_bound(dx, want, tol)
    for b, n in enumerate(lengths):
        assert (dx[b, max(n, 0):] == 0).all()


def test_backward_against_differences():
    """The gradient along a few directions against central differences of the
    oracle's loss: as far off as the elements' bounds allow, plus the
    differences' own error (h^2 times a third derivative of order 10)."""
    rng = np.random.default_rng(0)
    N, H, Hk, D, window, sinks = 40, 2, 1, 64, 9, 2
    x = rnd(rng, (1, N, (H + 2 * Hk) * D), 1.0, "float16")
    g = rnd(rng, (1, N, H * D), 0.5, "float16")
    out, lse = cu().dev_window_attention(up(x, "float16"), H, Hk, window, sinks, None, None, True)
    dx = down(cu().dev_window_attention_backward(up(g, "float16"), up(x, "float16"), out, lse, H, Hk, window, sinks))
    _, tol = backward_bound(g, x, H, Hk, window, sinks, D ** -0.5, "float16")
    h = 1e-4
    for _ in range(6):
        way = rng.standard_normal(x.shape)
        lo, hi = (ob.window_attention(x + s * way, H, Hk, window, sinks, D ** -0.5)[0] for s in (-h, h))
        num = ((hi - lo) * g).sum() / (2 * h)
        assert abs(num - (dx * way).sum()) < (tol * np.abs(way)).sum() + 1e-5


# ---- values at the top of the type ---------------------------------------------------

TOP = {"float16": 65504.0, "bfloat16": (2.0 - 2.0 ** -7) * 2.0 ** 127}


def top_values(rng, v, dtype):
    """v (..., D) with its last columns at the type's largest value, either sign."""
    v[..., -8:] = TOP[dtype] * np.where(np.arange(8) % 2, 1.0, -1.0)
    return v


def check_top(y, H, D, dtype):
    """An average of one number is that number (the bound of a sum over n keys, n
    below 2^14: under a quarter of a step)."""
    got = y.reshape(-1, H, D)[..., -8:]
    assert np.isfinite(got).all()
    assert (np.abs(got) >= TOP[dtype] * (1 - 2 * out_half_ulp_rel(dtype))).all()
    assert (np.sign(got) == np.where(np.arange(8) % 2, 1.0, -1.0)).all()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("N,H,D,window", [(333, 2, 64, None), (200, 3, 72, 50), (150, 2, 128, 90)])
def test_values_at_the_top_of_the_type(dtype, N, H, D, window):
    """The weights' rounding, or sums past the type's (or fp32's) largest value
    ahead of the division, may not make an average infinite."""
    rng = np.random.default_rng(N)
    x = rnd(rng, (1, N, (H + 2) * D), 1.0, dtype)
    x[..., :(H + 1) * D] *= 4.0
    top_values(rng, x[..., (H + 1) * D:], dtype)
    want, lse = ob.window_attention(x, H, 1, window, 2, 0.3)
    for with_lse in (False, True):
        y = cu().dev_window_attention(up(x, dtype), H, 1, window, 2, 0.3, None, with_lse)
        y = down(y[0] if with_lse else y)
        check_top(y, H, D, dtype)
        tol, _ = forward_bound(x, H, 1, window, 2, 0.3, dtype)
        check(y, want, tol, dtype)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("B,n,H,Hk,D,S", [(1, 1, 16, 2, 128, 5000), (2, 1, 8, 2, 72, 400), (3, 5, 4, 1, 64, 700), (1, 2, 4, 2, 96, 9000)])
def test_cached_values_at_the_top_of_the_type(dtype, B, n, H, Hk, D, S):
    rng = np.random.default_rng(S)
    q = rnd(rng, (B, n, H * D), 4.0, dtype)
    k, v = rnd(rng, (B, S, Hk * D), 1.0, dtype), rnd(rng, (B, S, Hk * D), 1.0, dtype)
    top_values(rng, v.reshape(B, S, Hk, D), dtype)
    y = down(cu().dev_window_attention_cached(up(q, dtype), up(k, dtype), up(v, dtype), ints([S - n] * B), H, Hk, None, 0,
                                              0.2))
    check_top(y, H, D, dtype)

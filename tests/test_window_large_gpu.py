"""Windowed attention on the kernels that large calls run (workgroups of 128
rows; split caches, merged or not), each at a size that chooses it, against
fp64."""
from __future__ import annotations

import numpy as np
import pytest

from helpers import check_bound, cu, down, out_half_ulp_rel, quantize, rnd, up
from test_window_gpu import check, check_top, ints, top_values
from window_cases import CACHED, LARGE, plan, rows64

pytestmark = pytest.mark.gpu


def whole(x, H, Hk, D, window, sinks, scale, dtype, lengths=None):
    """(out, bound, log-sums, bound): the weights are rounded once for their
    product with V (half a step each, and the sum they are divided by), scores
    carry D fp32 roundings (2^-23 a term of sum |q k|) plus a few steps of the
    exponent, both in the weights and their sum; check() adds the result's one
    rounding."""
    B, N, _ = x.shape
    h = x.astype(np.float64).reshape(B, N, H + 2 * Hk, D)
    out, tol = np.zeros((B, N, H, D)), np.zeros((B, N, H, D))
    lse, tl = np.full((B, H, N), -np.inf), np.zeros((B, H, N))
    for b in range(B):
        n = N if lengths is None else lengths[b]
        for a in range(H):
            u = a // (H // Hk)
            o, s, _, avg, size = rows64(h[b, :n, a], h[b, :n, H + u], h[b, :n, H + Hk + u], 0, window, sinks, scale)
            off = D * 2.0 ** -23 * abs(scale) * size
            out[b, :n, a], lse[b, a, :n] = o, s
            tol[b, :n, a] = (2 * out_half_ulp_rel(dtype) + 2 * (off[:, None] + 2.0 ** -18)) * avg
            tl[b, a, :n] = off + 2.0 ** -18 + 2.0 ** -22 * np.abs(s)
    return out.reshape(B, N, H * D), tol.reshape(B, N, H * D), lse, tl


def near_lse(got, lse, tl):
    none = np.isinf(lse)
    assert (np.isneginf(got) == none).all()
    check_bound(got[~none], lse[~none], tl[~none], "lse")


@pytest.mark.parametrize("dtype,B,N,H,Hk,D,window,sinks,lengths,launches", LARGE)
def test_forward_of_many_workgroups(dtype, B, N, H, Hk, D, window, sinks, lengths, launches):
    """With and without log-sums; NaN behind the lengths."""
    assert plan(B, H, Hk, N, 0, D, window, sinks) == launches
    rng = np.random.default_rng(N + D)
    x = rnd(rng, (B, N, (H + 2 * Hk) * D), 1.0, dtype)
    scale = 1.7 * D ** -0.5
    want, tol, lse, tl = whole(x, H, Hk, D, window, sinks, scale, dtype, lengths)
    for b, n in enumerate(lengths or []):
        x[b, n:] = np.nan
    gx, gn = up(x, dtype), None if lengths is None else ints(lengths)
    y, s = cu().dev_window_attention(gx, H, Hk, window, sinks, scale, gn, True)
    check(down(y), want, tol, dtype, "with lse")
    near_lse(down(s), lse, tl)
    plain = down(cu().dev_window_attention(gx, H, Hk, window, sinks, scale, gn))
    check(plain, want, tol, dtype)
    for b, n in enumerate(lengths or []):
        assert (plain[b, n:] == 0).all() and (down(y)[b, n:] == 0).all()
    assert (down(cu().dev_window_attention(gx, H, Hk, window, sinks, scale, gn)) == plain).all()


@pytest.mark.parametrize("D", [64, 72, 128])
@pytest.mark.parametrize("scale", [0.0, -0.3, 40.0])
def test_steep_rows_of_many_workgroups(D, scale):
    """Scores of hundreds, rising and falling along the keys: the references move
    far."""
    B, N, H = 9 if D == 64 else 5, 300, 12
    assert plan(B, H, 1, N, 0, D, 90, 5).startswith("window 128 rows")
    rng = np.random.default_rng(D)
    x = rnd(rng, (B, N, (H + 2) * D), 1.0, "bfloat16")
    x[:, :, H * D] = np.linspace(-2, 2, N)
    x = quantize(x, "bfloat16")
    want, tol, lse, tl = whole(x, H, 1, D, 90, 5, scale, "bfloat16")
    for with_lse in (False, True):
        y = cu().dev_window_attention(up(x, "bfloat16"), H, 1, 90, 5, scale, None, with_lse)
        if with_lse:
            y, s = y
            near_lse(down(s), lse, tl)
        check(down(y), want, tol, "bfloat16")


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("D", [64, 72, 128])
def test_values_that_rows_of_many_workgroups_do_not_see(D, value):
    """Value rows that are not finite, in both row blocks of a wave: the rows that
    see them are spoiled in that column, and no other."""
    B, N, H, window, sinks, dtype = 9 if D == 64 else 5, 300, 12, 40, 2, "bfloat16"
    assert plan(B, H, 1, N, 0, D, window, sinks).startswith("window 128 rows")
    rng = np.random.default_rng(D)
    x = rnd(rng, (B, N, (H + 2) * D), 1.0, dtype)
    column = (H + 1) * D + 7
    places = [3, 70, 150, 151, 299]  # 3: ahead of a window, past the sinks
    x[:, places, column] = 0.0
    want, tol, lse, tl = whole(x, H, 1, D, window, sinks, 0.125, dtype)
    x[:, places, column] = value
    i = np.arange(N)
    sees = np.zeros(N, bool)
    for at in places:
        sees |= (i >= at) & (i < at + window)
    for with_lse in (False, True):
        y = cu().dev_window_attention(up(x, dtype), H, 1, window, sinks, 0.125, None, with_lse)
        if with_lse:
            y, s = y
            near_lse(down(s), lse, tl)
        y = down(y).reshape(B, N, H, D)
        assert not np.isfinite(y[:, sees][..., 7]).any()
        y[:, sees, :, 7] = want.reshape(B, N, H, D)[:, sees, :, 7]
        check(y.reshape(B, N, H * D), want, tol, dtype)
    # a key that is not finite makes the scores of the rows that see it NaN
    x[:, places, column] = 0.0
    x[:, 150, H * D:(H + 1) * D] = np.nan
    sees = (i >= 150) & (i < 150 + window)
    y = down(cu().dev_window_attention(up(x, dtype), H, 1, window, sinks, 0.125)).reshape(B, N, H, D)
    assert np.isnan(y[:, sees]).all()
    w, t = want.reshape(B, N, H, D)[:, ~sees], tol.reshape(B, N, H, D)[:, ~sees]
    check(y[:, ~sees], w, t, dtype)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("D", [64, 96, 128])
def test_values_at_the_top_of_the_type_in_many_workgroups(dtype, D):
    B, N, H = 9 if D == 64 else 5, 300, 12
    assert plan(B, H, 1, N, 0, D, 130, 2).startswith("window 128 rows")
    rng = np.random.default_rng(D)
    x = rnd(rng, (B, N, (H + 2) * D), 1.0, dtype)
    x[..., :(H + 1) * D] *= 4.0
    top_values(rng, x[..., (H + 1) * D:], dtype)
    for with_lse in (False, True):
        y = cu().dev_window_attention(up(x, dtype), H, 1, 130, 2, 0.3, None, with_lse)
        check_top(down(y[0] if with_lse else y), H, D, dtype)


# ---- over a cache ------------------------------------------------------------------

def over_cache(q, k, v, lengths, H, Hk, window, sinks, scale, dtype):
    B, n, C = q.shape
    D, S = C // H, k.shape[1]
    out, tol = np.zeros((B, n, H, D)), np.zeros((B, n, H, D))
    for b in range(B):
        keys = min(lengths[b] + n, S)
        kb, vb = (a[b, :keys].reshape(keys, Hk, D) for a in (k, v))
        for a in range(H):
            u = a // (H // Hk)
            o, _, _, avg, size = rows64(q[b].reshape(n, H, D)[:, a], kb[:, u], vb[:, u], lengths[b], window, sinks, scale)
            out[b, :, a] = o
            tol[b, :, a] = (2 * out_half_ulp_rel(dtype) + 2 * (D * 2.0 ** -23 * abs(scale) * size[:, None] + 2.0 ** -18)) * avg
    return out.reshape(B, n, C), tol.reshape(B, n, C)


@pytest.mark.parametrize("dtype,B,n,H,Hk,D,S,window,sinks,launches", CACHED)
def test_caches(dtype, B, n, H, Hk, D, S, window, sinks, launches):
    """Lengths from none to the whole cache; what lies behind the new tokens is
    NaN, and so is a value that some or all of the new tokens' windows have just
    left: it spoils what sees it and nothing else."""
    assert plan(B, H, Hk, n, S, D, window, sinks) == launches
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
    scale = 1.3 * D ** -0.5
    want, tol = over_cache(q, k, v, lengths, H, Hk, window, sinks, scale, dtype)
    gq, gk, gn = up(q, dtype), up(k, dtype), ints(lengths)
    y = down(cu().dev_window_attention_cached(gq, gk, up(v, dtype), gn, H, Hk, window, sinks, scale))
    check(y, want, tol, dtype)
    if window is None:
        return
    reached = False
    for gone in sorted({1, n}):  # windows of the last n - gone + 1 tokens have left it
        bad, spoiled = v.copy(), np.zeros((B, n), bool)
        for b in range(B):
            at = lengths[b] + gone - 1 - window
            if at >= sinks:
                bad[b, at] = np.nan
                pos = lengths[b] + np.arange(n)
                spoiled[b] = (pos >= at) & (pos < at + window)
                reached = True
        y = down(cu().dev_window_attention_cached(gq, gk, up(bad, dtype), gn, H, Hk, window, sinks, scale))
        assert np.isnan(y[spoiled]).all()
        check(y[~spoiled], want[~spoiled], tol[~spoiled], dtype)
    assert reached


@pytest.mark.parametrize("dtype,B,n,H,Hk,D,S,window,sinks,launches", CACHED)
def test_caches_at_the_top_of_the_type(dtype, B, n, H, Hk, D, S, window, sinks, launches):
    rng = np.random.default_rng(S)
    q = rnd(rng, (B, n, H * D), 4.0, dtype)
    k, v = rnd(rng, (B, S, Hk * D), 1.0, dtype), rnd(rng, (B, S, Hk * D), 1.0, dtype)
    top_values(rng, v.reshape(B, S, Hk, D), dtype)
    y = down(cu().dev_window_attention_cached(up(q, dtype), up(k, dtype), up(v, dtype), ints([S - n] * B), H, Hk, window,
                                              sinks, 0.2))
    check_top(y, H, D, dtype)


# ---- gradients of many key blocks ----------------------------------------------------

def gradients(g, x, H, Hk, D, window, sinks, scale, dtype, lengths=None):
    """(dx, bound), the bound as test_window_gpu's: P and dS rounded once for their
    products, delta and the log-sums within another half step of the magnitudes,
    the scores' D fp32 roundings, sums of up to N rows of every head 2^-23 a term,
    the result's rounding; fp16's smallest steps of dS (2^-24)."""
    B, N, _ = x.shape
    h, gh = x.astype(np.float64).reshape(B, N, H + 2 * Hk, D), g.astype(np.float64).reshape(B, N, H, D)
    out, mag = np.zeros(h.shape), np.zeros(h.shape)
    for b in range(B):
        n = N if lengths is None else lengths[b]
        for a in range(H):
            u, v = H + a // (H // Hk), H + Hk + a // (H // Hk)
            qh, kh, vh, go = h[b, :n, a], h[b, :n, u], h[b, :n, v], gh[b, :n, a]
            o, _, p, avg, _ = rows64(qh, kh, vh, 0, window, sinks, scale)
            ds = p * (go @ vh.T - (go * o).sum(1, keepdims=True)) * scale
            size = p * (np.abs(go) @ np.abs(vh).T + (np.abs(go) * avg).sum(1, keepdims=True)) * abs(scale)
            for t, e, f in ((out, ds, lambda z: z), (mag, size, np.abs)):
                t[b, :n, a] = e @ f(kh)
                t[b, :n, u] += e.T @ f(qh)
                t[b, :n, v] += p.T @ f(go)
    hu = out_half_ulp_rel(dtype)
    most = np.abs(h[:, :, :H]).sum(-1).max() * np.abs(h[:, :, H:H + Hk]).max()
    rel = 3 * hu + 4 * D * 2.0 ** -23 * abs(scale) * most + (N * H // Hk + D) * 2.0 ** -23 + 2.0 ** -16
    tiny = 2.0 ** -24 * N * (H // Hk) * np.abs(x).max() * max(abs(scale), 1.0) if dtype == "float16" else 0.0
    tol = rel * mag + tiny
    return out.reshape(x.shape), (tol + hu * (np.abs(out) + tol) + 2.0 ** -24).reshape(x.shape)


@pytest.mark.parametrize("dtype,B,N,H,Hk,D,window,sinks,ragged", [
    ("bfloat16", 40, 300, 4, 4, 64, 100, 3, True), ("float16", 70, 130, 4, 2, 72, None, 0, True),
    ("bfloat16", 2, 1100, 16, 4, 128, 300, 70, False), ("float16", 3, 700, 12, 3, 96, 2, 640, False),
])
def test_gradients_of_many_key_blocks(dtype, B, N, H, Hk, D, window, sinks, ragged):
    """More key blocks than the plan's workgroup has threads, as many ranges as
    CUs, key blocks cut into many ranges."""
    rng = np.random.default_rng(N)
    x, g = rnd(rng, (B, N, (H + 2 * Hk) * D), 1.0, dtype), rnd(rng, (B, N, H * D), 0.5, dtype)
    lengths = None
    if ragged:
        lengths = rng.integers(0, N + 1, B)
        lengths[:3] = 0, N, 1
    want, tol = gradients(g, x, H, Hk, D, window, sinks, D ** -0.5, dtype, lengths)
    if ragged:
        for b, n in enumerate(lengths):
            x[b, n:], g[b, n:] = np.nan, np.nan
    gx, gg, gn = up(x, dtype), up(g, dtype), None if lengths is None else ints(lengths)
    out, lse = cu().dev_window_attention(gx, H, Hk, window, sinks, None, gn, True)
    args = gg, gx, out, lse, H, Hk, window, sinks, None, gn
    dx = down(cu().dev_window_attention_backward(*args))
    check_bound(dx, want, tol)
    assert (down(cu().dev_window_attention_backward(*args)) == dx).all()

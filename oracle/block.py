"""fp64 restatement of the causal block's operators: norms of queries and keys
with the rotation, windowed attention with sinks, gated feed-forward layers,
each with its gradients (test infrastructure; NumPy, no reference
counterpart)."""
from __future__ import annotations

import numpy as np

from oracle.experts import act, act_slope


# ---- norms and rotation -------------------------------------------------------

def rope_table(length, columns, base=10000.0):
    turn = np.array([[p * base ** (-2.0 * j / columns) for j in range(columns // 2)] for p in range(length)])
    return np.concatenate([np.cos(turn), np.sin(turn)], 1)


def pairs_of(R, interleaved):
    """The two columns of pair j."""
    return [(2 * j, 2 * j + 1) if interleaved else (j, j + R // 2) for j in range(R // 2)]


def rotate(x, table, positions, interleaved, back=False):
    """x (B, N, heads, D) turned by the table's rows; a missing row gives NaN."""
    out = np.array(x, np.float64)
    if table is None:
        return out
    R = table.shape[1]
    rows = np.full(positions.shape + (R,), np.nan)
    ok = (positions >= 0) & (positions < len(table))
    rows[ok] = table[positions[ok]]
    for j, (a, b) in enumerate(pairs_of(R, interleaved)):
        c, s = rows[:, :, None, j], rows[:, :, None, R // 2 + j]
        if back:
            s = -s
        out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return out


def norm(x, kind, eps):
    """(hat, r) over the last axis."""
    x = np.asarray(x, np.float64)
    if kind == "layer":
        x = x - x.mean(-1, keepdims=True)
    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    return x * r, r


def of_heads(p, H, Hk, D, fill):
    """A (2, D) parameter spread over the query and key heads."""
    if p is None:
        return np.full((H + Hk, D), fill, np.float64)
    p = np.asarray(p, np.float64)
    return np.concatenate([np.repeat(p[:1], H, 0), np.repeat(p[1:], Hk, 0)])


def qk_norm_rope(x, H, Hk, table, positions, weight=None, bias=None, kind="rms", eps=1e-6, interleaved=False):
    """(B, N, (H + 2 Hk) D) -> the same shape; and the magnitude its fp32
    rounding errors scale with."""
    B, N, C = x.shape
    D = C // (H + 2 * Hk)
    h = np.asarray(x, np.float64).reshape(B, N, H + 2 * Hk, D)
    qk = h[:, :, :H + Hk]
    hat, r = norm(qk, kind, eps)
    w, b = of_heads(weight, H, Hk, D, 1.0), of_heads(bias, H, Hk, D, 0.0)
    y = rotate(hat * w + b, table, positions, interleaved)
    size = np.abs(qk) + (np.abs(qk.mean(-1, keepdims=True)) if kind == "layer" else 0.0)
    mag = size * r * np.abs(w) + np.abs(b)
    if table is not None:
        for i, j in pairs_of(table.shape[1], interleaved):
            mag[..., i] = mag[..., j] = mag[..., i] + mag[..., j]
    v = h[:, :, H + Hk:]
    return (np.concatenate([y, v], 2).reshape(B, N, C), np.concatenate([mag, np.zeros_like(v)], 2).reshape(B, N, C))


def qk_norm_rope_backward(g, x, H, Hk, table, positions, weight=None, kind="rms", eps=1e-6, interleaved=False):
    """(dx, dweight, dbias), and the magnitudes of their errors."""
    B, N, C = x.shape
    D = C // (H + 2 * Hk)
    gh = np.asarray(g, np.float64).reshape(B, N, H + 2 * Hk, D)
    qk = np.asarray(x, np.float64).reshape(B, N, H + 2 * Hk, D)[:, :, :H + Hk]
    hat, r = norm(qk, kind, eps)
    w = of_heads(weight, H, Hk, D, 1.0)
    d = rotate(gh[:, :, :H + Hk], table, positions, interleaved, back=True)
    e = d * w
    dx = e - hat * (e * hat).mean(-1, keepdims=True)
    if kind == "layer":
        dx = dx - e.mean(-1, keepdims=True)
    dx = dx * r
    sums = [(d * hat).sum((0, 1)), d.sum((0, 1))]
    dw, db = (np.stack([s[:H].sum(0), s[H:].sum(0)]) for s in sums)
    am = np.abs(gh[:, :, :H + Hk]).copy()
    if table is not None:
        for i, j in pairs_of(table.shape[1], interleaved):
            am[..., i] = am[..., j] = am[..., i] + am[..., j]
    size = (np.abs(qk) + (np.abs(qk.mean(-1, keepdims=True)) if kind == "layer" else 0.0)) * r
    ae = am * np.abs(w)
    mx = r * (ae + size * (ae * size).mean(-1, keepdims=True) + ae.mean(-1, keepdims=True))
    v = gh[:, :, H + Hk:]
    mags = [(am * size).sum((0, 1)), am.sum((0, 1))]
    mw, mb = (np.stack([s[:H].sum(0), s[H:].sum(0)]) for s in mags)
    return ((np.concatenate([dx, v], 2).reshape(B, N, C), dw, db),
            (np.concatenate([mx, np.zeros_like(v)], 2).reshape(B, N, C), mw, mb))


# ---- gated feed-forward -------------------------------------------------------

def gate_act(v, kind):
    return v if kind is None else act(v, kind)


def gate_slope(v, kind):
    return np.ones_like(v) if kind is None else act_slope(v, kind)


def gated(x, W, b, kind):
    """(y, pre), and the products' sums of magnitudes (for either projection)."""
    x, W = np.asarray(x, np.float64), np.asarray(W, np.float64)
    F = len(W) // 2
    pre = x @ W.T + (0.0 if b is None else np.asarray(b, np.float64))
    mag = np.abs(x) @ np.abs(W).T + (0.0 if b is None else np.abs(b))
    return gate_act(pre[:, :F], kind) * pre[:, F:], pre, mag


def gated_backward(g, x, W, pre, kind):
    """(dx, dW, db, dpre)."""
    g, x, W, pre = (np.asarray(a, np.float64) for a in (g, x, W, pre))
    F = len(W) // 2
    gate, up = pre[:, :F], pre[:, F:]
    d = np.concatenate([g * up * gate_slope(gate, kind), g * gate_act(gate, kind)], 1)
    return d @ W, d.T @ x, d.sum(0), d


# ---- windowed attention -------------------------------------------------------

def visible(i, j, window, sinks):
    """Whether the query at position i sees the key at position j."""
    return j <= i and (window is None or j > i - window or j < sinks)


def window_rows(q, k, v, first, window, sinks, scale):
    """One head: queries at positions first .. first + n - 1 over keys 0 ..
    len(k) - 1.  (out, lse, weights); a row without a key gives 0 and -inf."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    n, S = len(q), len(k)
    out, lse, p = np.zeros((n, v.shape[1])), np.full(n, -np.inf), np.zeros((n, S))
    for i in range(n):
        at = np.array([j for j in range(S) if visible(first + i, j, window, sinks)], np.int64)
        if not len(at):
            continue
        s = scale * (k[at] @ q[i])
        m = s.max()
        e = np.exp(s - m)
        p[i, at] = e / e.sum()
        lse[i] = m + np.log(e.sum())
        out[i] = p[i, at] @ v[at]
    return out, lse, p


def split_heads(x, H, Hk):
    B, N, C = x.shape
    D = C // (H + 2 * Hk)
    h = np.asarray(x, np.float64).reshape(B, N, H + 2 * Hk, D)
    return h[:, :, :H], h[:, :, H:H + Hk], h[:, :, H + Hk:]


def window_attention(x, H, Hk, window, sinks, scale, lengths=None):
    """(out (B, N, H D), lse (B, H, N)) of a packed projection."""
    q, k, v = split_heads(x, H, Hk)
    B, N, _, D = q.shape
    out, lse = np.zeros((B, N, H, D)), np.full((B, H, N), -np.inf)
    for b in range(B):
        n = N if lengths is None else min(max(int(lengths[b]), 0), N)
        for h in range(H):
            u = h // (H // Hk)
            out[b, :n, h], lse[b, h, :n], _ = window_rows(q[b, :n, h], k[b, :n, u], v[b, :n, u], 0, window, sinks, scale)
    return out.reshape(B, N, H * D), lse


def window_attention_backward(g, x, H, Hk, window, sinks, scale, lengths=None):
    """The packed gradient, and the sums of magnitudes its errors scale with."""
    q, k, v = split_heads(x, H, Hk)
    B, N, _, D = q.shape
    g = np.asarray(g, np.float64).reshape(B, N, H, D)
    out, mag = np.zeros((B, N, H + 2 * Hk, D)), np.zeros((B, N, H + 2 * Hk, D))
    for b in range(B):
        n = N if lengths is None else min(max(int(lengths[b]), 0), N)
        for h in range(H):
            u = h // (H // Hk)
            qh, kh, vh, gh = q[b, :n, h], k[b, :n, u], v[b, :n, u], g[b, :n, h]
            o, _, p = window_rows(qh, kh, vh, 0, window, sinks, scale)
            dp = gh @ vh.T
            ds = p * (dp - (gh * o).sum(1, keepdims=True)) * scale
            size = p * (np.abs(gh) @ np.abs(vh).T + (np.abs(gh) * (p @ np.abs(vh))).sum(1, keepdims=True)) * scale
            out[b, :n, h] = ds @ kh
            out[b, :n, H + u] += ds.T @ qh
            out[b, :n, H + Hk + u] += p.T @ gh
            mag[b, :n, h] = size @ np.abs(kh)
            mag[b, :n, H + u] += size.T @ np.abs(qh)
            mag[b, :n, H + Hk + u] += p.T @ np.abs(gh)
    return out.reshape(x.shape), mag.reshape(x.shape)


def window_attention_cached(q, k, v, lengths, H, Hk, window, sinks, scale):
    """q (B, n, H D) at positions lengths[b] + i over caches (B, S, Hk D)."""
    B, n, C = q.shape
    D, S = C // H, k.shape[1]
    out = np.zeros((B, n, H, D))
    for b in range(B):
        first = int(lengths[b])
        keys = min(first + n, S)
        for h in range(H):
            u = h // (H // Hk)
            kb, vb = (np.asarray(a, np.float64)[b, :keys].reshape(keys, Hk, D)[:, u] for a in (k, v))
            out[b, :, h], _, _ = window_rows(np.asarray(q, np.float64)[b].reshape(n, H, D)[:, h], kb, vb, first, window,
                                             sinks, scale)
    return out.reshape(B, n, C)

"""fp64 restatement of the expert operators: routing, the row exchange and
products over ragged groups (test infrastructure; NumPy loops, no reference
counterpart)."""
from __future__ import annotations

import numpy as np


def route(logits, k, renormalize=True):
    """(weights, experts, offsets, slots) of logits (T, E), chosen one token at
    a time: the k largest, equal ones by index, NaN above every number."""
    v = np.asarray(logits, np.float64)
    T, E = v.shape
    weights, experts = np.zeros((T, k)), np.zeros((T, k), np.int64)
    for t in range(T):
        rank = sorted(range(E), key=lambda e: (0 if np.isnan(v[t, e]) else 1,
                                               0.0 if np.isnan(v[t, e]) else -v[t, e], e))[:k]
        experts[t] = rank
        top = v[t, rank[0]]
        if top == -np.inf:
            continue
        with np.errstate(invalid="ignore"):
            p = np.exp(v[t] - top)
        weights[t] = p[rank] / (p[rank].sum() if renormalize else p.sum())
    places = [(e, a) for a, e in enumerate(experts.reshape(-1))]
    slots = np.zeros(T * k, np.int64)
    for place, (_, a) in enumerate(sorted(places)):
        slots[a] = place
    offsets = np.array([sum(1 for e, _ in places if e < x) for x in range(E + 1)])
    return weights, experts, offsets, slots.reshape(T, k)


def route_weights(logits, experts, renormalize=True):
    """The weights of a given choice, differentiable in the logits."""
    v = np.asarray(logits, np.float64)
    p = np.exp(v - v.max(1, keepdims=True))
    w = np.take_along_axis(p, experts, 1)
    return w / (w if renormalize else p).sum(1, keepdims=True)


def route_backward(g, logits, experts, renormalize=True):
    """Gradient of the logits by the softmax rule over the experts that carry
    the normalisation."""
    v = np.asarray(logits, np.float64)
    out = np.zeros_like(v)
    for t in range(v.shape[0]):
        top = v[t].max()
        if top == -np.inf:
            continue
        over = sorted(experts[t]) if renormalize else range(v.shape[1])
        over = np.array(list(over))
        p = np.exp(v[t, over] - top)
        p /= p.sum()
        up = np.zeros(v.shape[1])
        up[experts[t]] = g[t]
        out[t, over] = p * (up[over] - (p * up[over]).sum())
    return out


def groups(offsets, rows):
    """(first, last) row of each group for any content of offsets."""
    out, end = [], 0
    for o in list(offsets)[1:]:
        nxt = max(end, min(max(int(o), 0), rows))
        out.append((end, nxt))
        end = nxt
    return out


def grouped_linear(x, w, offsets, bias=None):
    """(y, sum |x||w|): y[r] = W[e] x[r] + b[e], 0 for rows of no group."""
    x, w = np.asarray(x, np.float64), np.asarray(w, np.float64)
    y = np.zeros((x.shape[0], w.shape[1]))
    mag = np.zeros_like(y)
    for e, (lo, hi) in enumerate(groups(offsets, x.shape[0])):
        y[lo:hi] = x[lo:hi] @ w[e].T + (0.0 if bias is None else np.asarray(bias, np.float64)[e])
        mag[lo:hi] = np.abs(x[lo:hi]) @ np.abs(w[e]).T
    return y, mag


def grouped_linear_backward(g, x, w, offsets):
    """((dx, dw, db), their sums of magnitudes)."""
    g, x, w = (np.asarray(a, np.float64) for a in (g, x, w))
    dx, dw, db = np.zeros_like(x), np.zeros_like(w), np.zeros(w.shape[:2])
    mx, mw, mb = np.zeros_like(x), np.zeros_like(w), np.zeros(w.shape[:2])
    for e, (lo, hi) in enumerate(groups(offsets, x.shape[0])):
        dx[lo:hi], mx[lo:hi] = g[lo:hi] @ w[e], np.abs(g[lo:hi]) @ np.abs(w[e])
        dw[e], mw[e] = g[lo:hi].T @ x[lo:hi], np.abs(g[lo:hi]).T @ np.abs(x[lo:hi])
        db[e], mb[e] = g[lo:hi].sum(0), np.abs(g[lo:hi]).sum(0)
    return (dx, dw, db), (mx, mw, mb)


def act(v, name):
    v = np.asarray(v, np.float64)
    if name == "silu":
        return v / (1.0 + np.exp(-v))
    if name == "gelu":
        return 0.5 * v * (1.0 + np.tanh(np.sqrt(2.0 / np.pi) * (v + 0.044715 * v ** 3)))
    return v


def act_slope(v, name):
    v = np.asarray(v, np.float64)
    if name == "silu":
        s = 1.0 / (1.0 + np.exp(-v))
        return s + v * s * (1.0 - s)
    if name == "gelu":
        c = np.sqrt(2.0 / np.pi)
        t = np.tanh(c * (v + 0.044715 * v ** 3))
        return 0.5 * (1.0 + t) + 0.5 * v * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * v * v)
    return np.ones_like(v)


def q4_weight(q, scales, zeros=None):
    """The weight (..., N, K) that packed q (..., N, K / 2), scales (..., K /
    G, N) and zero points stand for."""
    q = np.asarray(q)
    w = np.zeros(q.shape[:-1] + (2 * q.shape[-1],))
    w[..., 0::2], w[..., 1::2] = q % 16, q // 16
    s = np.swapaxes(np.asarray(scales, np.float64), -1, -2)
    z = np.full(s.shape, 8.0) if zeros is None else np.swapaxes(np.asarray(zeros, np.float64), -1, -2)
    of = np.arange(w.shape[-1]) // (w.shape[-1] // s.shape[-1])
    return (w - z[..., of]) * s[..., of]

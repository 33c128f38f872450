"""Every variant of the 4-bit layer's kernel against fp64: all tiles and wave
counts, dense and per group of rows, every width of the scale groups, zero
points over the whole byte, scales that pass through LDS in several parts."""
from __future__ import annotations

import numpy as np
import pytest

from helpers import check_bound, cu, down, out_half_ulp_rel, rnd, up
from oracle import experts as ox
from q4_cases import PARTS, plan, variant_cases

pytestmark = pytest.mark.gpu


def raw(a, dtype):
    return cu().gputensor_from_numpy(np.ascontiguousarray(a, dtype))


def walk_bound(x, s, y, dtype, act, top):
    """For independent random terms.  The kernel's sums run over x (16 + q) s
    and take (16 + z) x s out again, `top` x s at most each: the 2 K fp32
    roundings are a random walk, and 64 sqrt(2 K) 2^-24 of the terms' 2-norm
    covers six standard deviations of it ten times over.  Then one rounding
    (half an ulp) of the result; activations have slopes of at most 1.13."""
    K, KG = x.shape[1], s.shape[0]
    squares = (x.astype(np.float64) ** 2).reshape(len(x), KG, K // KG).sum(2) @ s.astype(np.float64) ** 2
    walk = 64 * 2.0 ** -24 * np.sqrt(2 * K) * top * np.sqrt(squares)
    return (1.2 if act else 1.0) * walk + (out_half_ulp_rel(dtype) + 2e-6) * np.abs(y) + 1e-7


def check(R, E, N, K, G, zeros, dtype, act, most):
    """y of R rows in E groups (0: one weight) against the formula at every row
    and 192 columns: the tiles' edges, the last ones and others."""
    g = cu()
    rng = np.random.default_rng(R + N + K + G)
    lead = (E,) if E else ()
    x = rnd(rng, (R, K), 1.0, dtype)
    q = rng.integers(0, 256, lead + (N, K // 2), dtype=np.uint8)
    s = np.abs(rnd(rng, lead + (K // G, N), 0.01, dtype))
    z = rng.integers(0, most + 1, s.shape, dtype=np.uint8) if zeros else None
    b = rnd(rng, lead + (N,), 1.0, dtype)
    off = np.concatenate([[0], np.sort(rng.integers(0, R + 1, E))]) if E else np.array([0, R])
    got = down(g.dev_linear_q4(up(x, dtype), raw(q, np.uint8), up(s, dtype), None if z is None else raw(z, np.uint8),
                               up(b, dtype), act, raw(off, np.int32) if E else None))
    assert got.shape == (R, N) and np.isfinite(got).all() and (got[off[-1]:] == 0).all()
    cols = np.unique(np.concatenate([[0, 15, 16, 31, 32, 63, 64, N - 1, N - 2, N // 16 * 16, N // 64 * 64],
                                     rng.integers(0, N, 192)]).clip(0, N - 1))
    for e in range(max(1, E)):
        at = (e,) if E else ()
        xe = x[off[e]:off[e + 1]]
        if not len(xe):
            continue
        se = s[at][:, cols]
        w = ox.q4_weight(q[at][cols], se, None if z is None else z[at][:, cols])
        y = ox.act(xe.astype(np.float64) @ w.T + b[at][cols], act)
        check_bound(got[off[e]:off[e + 1]][:, cols], y, walk_bound(xe, se, y, dtype, act, 16 + max(15, most)),
                    "group %d" % e)


def the_card_is_whole():
    return cu().get_device_properties(0)["multi_processor_count"] == 256


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("i,case", list(enumerate(variant_cases())))
def test_variant(i, case, dtype):
    R, E, N, K, G, zeros, cols, waves = case
    if the_card_is_whole():
        assert plan(R, E, N, K, G, zeros).startswith("q4 16x%d %d waves," % (cols, waves))
    check(R, E, N, K, G, zeros, dtype, (None, "silu", "gelu")[i % 3], 255 if zeros else 8)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("R,E,N,K,G,zeros,parts", PARTS)
def test_scales_in_parts(dtype, R, E, N, K, G, zeros, parts):
    if the_card_is_whole():
        assert plan(R, E, N, K, G, zeros).endswith("scales in %d" % parts)
    check(R, E, N, K, G, zeros, dtype, None, 15 if zeros else 8)

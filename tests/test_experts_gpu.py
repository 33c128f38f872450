"""Expert operators on the GPU against the fp64 oracle."""
from __future__ import annotations

import ctypes
import os

import numpy as np
import pytest

from helpers import check_bound, cu, down, gemm_bound, out_half_ulp_rel, quantize, rnd, up
from oracle import experts as ox

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
I64, P = ctypes.c_int64, ctypes.c_void_p
SFD = {"float32": 0, "float16": 1, "bfloat16": 2}
DTYPES = ["float32", "float16", "bfloat16"]


def ints(a):
    return cu().gputensor_from_numpy(np.ascontiguousarray(a, np.int32))


def f32(a):
    return cu().gputensor_from_numpy(np.ascontiguousarray(a, np.float32))


def raw(gt):
    return cu().gputensor_to_numpy(gt)


# ---- routing ------------------------------------------------------------------

def logits(rng, T, E, dtype, masked=False):
    v = quantize((rng.standard_normal((T, E)) * 2).astype(np.float32), dtype)
    if masked:
        v[rng.random((T, E)) < 0.6] = -np.inf
        v[::5] = -np.inf
    return v


def weight_bound(v, w):
    """fp32 softmax weights: the exponent's argument is rounded once (half a
    step of at most |d| = max - v), exp and the division are a few steps each,
    and the sum's E roundings act on positive terms."""
    finite = np.where(np.isfinite(v), v, 0.0)
    spread = (finite.max(1) - finite.min(1))[:, None]
    return (spread + v.shape[1] + 16) * 2.0 ** -24 * w + 1e-37


@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("dtype,T,E,k,masked", [
    ("float32", 1, 1, 1, False), ("float32", 1, 2, 1, False), ("bfloat16", 16, 8, 2, False),
    ("float16", 64, 64, 8, True), ("bfloat16", 65, 65, 8, False), ("float32", 700, 60, 4, True),
    ("bfloat16", 1000, 7, 7, True), ("float32", 130, 300, 16, False), ("float16", 67, 1024, 3, True),
])
def test_route(dtype, T, E, k, masked, renorm):
    g = cu()
    rng = np.random.default_rng(T + E)
    v = logits(rng, T, E, dtype, masked)
    w, e, off, slots = ox.route(v, k, renorm)
    lt = up(v, dtype)
    got = g.dev_route_topk(lt, k, renorm)
    assert np.array_equal(raw(got[1]), e)
    assert np.array_equal(raw(got[2]), off)
    assert np.array_equal(raw(got[3]), slots)
    check_bound(raw(got[0]), w, weight_bound(v, w), "weights")
    gr = rng.standard_normal((T, k)).astype(np.float32)
    d = ox.route_backward(gr, v, e, renorm)
    dl = down(g.dev_route_topk_backward(f32(gr), lt, got[0], got[1], renorm))
    # w (g - <g, w>): the weights' own error twice, and k + 2 roundings of
    # terms no larger than the largest gradient's
    big = np.abs(gr).max(1, keepdims=True)
    p = np.zeros((T, E)) if renorm else ox.route(v, E, False)[0][:, :0]
    if renorm:
        np.put_along_axis(p, e, w, 1)
    else:
        p = np.where(np.isfinite(v).any(1, keepdims=True), np.exp(np.where(np.isfinite(v), v, -np.inf) - np.where(
            np.isfinite(v).any(1, keepdims=True), v.max(1, keepdims=True), 0)), 0)
        s = p.sum(1, keepdims=True)
        p = p / np.where(s == 0, 1, s)
    bound = 4 * big * (weight_bound(v, p) + (k + 4) * 2.0 ** -24 * p)
    check_bound(dl, d, bound + out_half_ulp_rel(dtype) * np.abs(d) + 2.0 ** -25, "logits' gradient")


@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("T,E,k,masked", [(90, 100, 6, False), (70, 128, 4, True), (200, 129, 8, True), (66, 256, 16, False), (130, 700, 5, True)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_route_many_experts(dtype, T, E, k, masked, renorm):
    """Two, four and sixteen logits a lane, in every type."""
    test_route(dtype, T, E, k, masked, renorm)


def test_route_ties_nan_and_infinities():
    g = cu()
    v = np.array([[3, 3, 3, 3], [-0.0, 0.0, -0.0, 0.0], [np.nan, 1, np.nan, 2], [np.inf, 1, 2, np.inf],
                  [-np.inf, -np.inf, 1, -np.inf], [-3.4e38, -3.4e38, -3.4e38, -3.4e38],
                  [-np.inf, -np.inf, -np.inf, -np.inf], [-np.inf, 1, -np.inf, 5]], np.float32)
    w, e, off, slots = (raw(t) for t in g.dev_route_topk(up(v, "float32"), 3))
    assert e.tolist() == [[0, 1, 2], [0, 1, 2], [0, 2, 3], [0, 3, 2], [2, 0, 1], [0, 1, 2], [0, 1, 2], [3, 1, 0]]
    third = np.float32(1) / np.float32(3)
    assert np.allclose(w[[0, 1, 5]], third, rtol=2e-7) and np.isnan(w[2]).all() and np.isnan(w[3]).any()
    assert w[4].tolist() == [1, 0, 0] and w[6].tolist() == [0, 0, 0] and w[7, 2] == 0
    assert off[-1] == 24 and sorted(slots.reshape(-1).tolist()) == list(range(24))
    d = raw(g.dev_route_topk_backward(f32(np.ones((8, 3))), up(v, "float32"), f32(w), ints(e)))
    assert (d[6] == 0).all() and (d[4] == 0).all()


@pytest.mark.parametrize("T,E,k", [(32768, 5, 1), (40001, 37, 3), (33000, 1000, 2)])
def test_route_many_tokens(T, E, k):
    """More blocks than are summed by every block: places and offsets exact."""
    g = cu()
    v = rnd(np.random.default_rng(T), (T, E), 1.0, "bfloat16")
    w, e, off, slots = (raw(t) for t in g.dev_route_topk(up(v, "bfloat16"), k))
    want = np.argsort(-v.astype(np.float64), axis=1, kind="stable")[:, :k]
    assert np.array_equal(e, want)
    flat = want.reshape(-1)
    place = np.empty(T * k, np.int64)
    place[np.argsort(flat, kind="stable")] = np.arange(T * k)
    assert np.array_equal(slots.reshape(-1), place)
    assert np.array_equal(off, np.concatenate([[0], np.bincount(flat, minlength=E).cumsum()]))
    assert np.allclose(w.sum(1), 1, atol=1e-6)


@pytest.mark.parametrize("act,code", [("silu", 4), ("gelu", 5)])
def test_activation_slopes_far_out(act, code):
    g = cu()
    lib = ctypes.CDLL(os.path.join(ROOT, "scaffolding_amd", "libsfgemm.so"))
    v = np.array([0.0, -0.0, 1e-30, 5, -5, 9.9, -9.9, 10.1, -10.1, 30, -30, 79, -79, 81, -81, 1e30, -1e30, np.inf, -np.inf,
                  np.nan], np.float32)
    a, b = f32(np.ones_like(v)), f32(v)
    out = g.empty(v.shape)
    assert lib.sf_act_backward(P(a.data_ptr), P(b.data_ptr), P(out.data_ptr), I64(v.size), 0, code, None) == 0
    got = raw(out)
    fin = v[:-3].astype(np.float64)
    with np.errstate(over="ignore", under="ignore", invalid="ignore"):
        want = np.where(np.abs(fin) > 100, fin > 0, ox.act_slope(np.clip(fin, -100, 100), act))
    # the exponential's argument is off by a few steps of |x| (c0 + c1 x^2 at gelu)
    assert (np.abs(got[:-3] - want) <= 200 * 2.0 ** -24 * np.abs(want) + 4e-7).all()
    assert got[-3] == 1 and abs(got[-2]) < 1e-30 and np.isnan(got[-1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 7, 2049, 2048 * 300 + 5])
def test_activation_slopes_in_place(dtype, n):
    """The result over the gradient or over the layer's output: the same bits
    as into memory of its own."""
    g = cu()
    lib = ctypes.CDLL(os.path.join(ROOT, "scaffolding_amd", "libsfgemm.so"))
    rng = np.random.default_rng(n)
    gr, pre = rnd(rng, (n,), 1.0, dtype), rnd(rng, (n,), 3.0, dtype)

    def run(into, code):
        t = [up(gr, dtype), up(pre, dtype), g.empty((n,), up(gr, dtype).dtype)]
        assert lib.sf_act_backward(P(t[0].data_ptr), P(t[1].data_ptr), P(t[into].data_ptr), I64(n), SFD[dtype], code,
                                   None) == 0
        return down(t[into])

    for act, code in (("silu", 4), ("gelu", 5)):
        own = run(2, code)
        want = gr.astype(np.float64) * ox.act_slope(pre, act)
        check_bound(own, want, out_half_ulp_rel(dtype) * np.abs(want) + 16 * 4 * 2.0 ** -24 * np.abs(gr) + 2.0 ** -25)
        assert np.array_equal(run(0, code), own) and np.array_equal(run(1, code), own)


def test_route_no_tokens_and_leading_shapes():
    g = cu()
    w, e, off, slots = g.dev_route_topk(g.empty((0, 5)), 2)
    assert raw(off).tolist() == [0] * 6 and w.shape == (0, 2) and slots.shape == (0, 2)
    assert g.dev_route_topk_backward(g.empty((0, 2)), g.empty((0, 5)), w, e).shape == (0, 5)
    v = rnd(np.random.default_rng(0), (3, 5, 7), 1.0, "float32")
    w, e, off, slots = g.dev_route_topk(up(v, "float32"), 2)
    assert w.shape == (3, 5, 2) and np.array_equal(raw(e).reshape(15, 2), ox.route(v.reshape(15, 7), 2)[1])


# ---- rows between token order and expert order -----------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,D", [(1, 1, 1), (5, 3, 7), (33, 2, 8), (9, 8, 65), (17, 2, 513), (40, 2, 1283),
                                   (3, 16, 2048), (70, 1, 4096), (2, 5, 8201)])
def test_row_exchange(dtype, T, k, D):
    g = cu()
    rng = np.random.default_rng(T * D)
    x, y, gr = (rnd(rng, s, 1.0, dtype) for s in ((T, D), (T * k, D), (T, D)))
    w = rng.random((T, k)).astype(np.float32)
    slots = rng.permutation(T * k).reshape(T, k)
    xt, yt, gt, wt, st = up(x, dtype), up(y, dtype), up(gr, dtype), f32(w), ints(slots)
    rows = down(g.dev_dispatch_rows(xt, st))
    want = np.zeros((T * k, D), np.float32)
    for j in range(k):
        want[slots[:, j]] = x
    assert np.array_equal(rows, want)
    for ww, tt in ((w, wt), (np.ones_like(w), None)):
        terms = ww.astype(np.float64)[:, :, None] * y.astype(np.float64)[slots]
        check_bound(down(g.dev_combine_rows(yt, st, tt)), terms.sum(1),
                    k * 2.0 ** -24 * np.abs(terms).sum(1) + out_half_ulp_rel(dtype) * (
                        1 + k * 2.0 ** -23) * np.abs(terms.sum(1)) + 2.0 ** -25, "combine")
    dy, dw = g.dev_combine_rows_backward(gt, yt, st, wt)
    want = np.zeros((T * k, D))
    for j in range(k):
        want[slots[:, j]] = w[:, j, None].astype(np.float64) * gr
    check_bound(down(dy), want, (out_half_ulp_rel(dtype) + 2.0 ** -23) * np.abs(want) + 2.0 ** -25, "rows' gradient")
    prod = gr.astype(np.float64)[:, None, :] * y.astype(np.float64)[slots]
    check_bound(raw(dw), prod.sum(2), D * 2.0 ** -24 * np.abs(prod).sum(2) + 1e-30, "weights' gradient")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,D", [(4095, 3, 72), (4096, 1, 1), (4096, 8, 500), (4096, 2, 512), (4099, 3, 513),
                                   (4099, 8, 331), (5000, 2, 1283), (4200, 1, 2056)])
def test_row_exchange_gradient_of_many_tokens(dtype, T, k, D):
    """Tokens enough to fill the GPU: a wave a token, its slots in turn, rows
    within a wave's columns and past them."""
    g = cu()
    rng = np.random.default_rng(T * D)
    y, gr = rnd(rng, (T * k, D), 1.0, dtype), rnd(rng, (T, D), 1.0, dtype)
    w = rng.random((T, k)).astype(np.float32)
    slots = rng.permutation(T * k).reshape(T, k)
    dy, dw = g.dev_combine_rows_backward(up(gr, dtype), up(y, dtype), ints(slots), f32(w))
    dy, dw = down(dy), raw(dw)
    for j in range(k):
        want = w[:, j, None].astype(np.float64) * gr
        check_bound(dy[slots[:, j]], want, (out_half_ulp_rel(dtype) + 2.0 ** -23) * np.abs(want) + 2.0 ** -25, "rows")
        prod = gr.astype(np.float64) * y[slots[:, j]]
        check_bound(dw[:, j], prod.sum(1), D * 2.0 ** -24 * np.abs(prod).sum(1) + 1e-30, "weights")


def test_row_exchange_empty_and_skipped():
    g = cu()
    assert g.dev_dispatch_rows(g.empty((0, 8)), ints(np.zeros((0, 2)))).shape == (0, 8)
    assert g.dev_combine_rows(g.empty((4, 0)), ints([[0, 1], [2, 3]])).shape == (2, 0)
    dy, dw = g.dev_combine_rows_backward(g.empty((2, 0)), g.empty((4, 0)), ints([[0, 1], [2, 3]]), f32(np.ones((2, 2))))
    assert (raw(dw) == 0).all()
    # slots out of range are skipped, and nothing is read or written there
    y = rnd(np.random.default_rng(0), (4, 24), 1.0, "float32")
    st = ints([[0, -1], [4, 2 ** 31 - 1]])
    out = raw(g.dev_combine_rows(up(y, "float32"), st))
    assert np.array_equal(out[0], y[0]) and (out[1] == 0).all()
    _, dw = g.dev_combine_rows_backward(f32(np.ones((2, 24))), up(y, "float32"), st, f32(np.ones((2, 2))))
    assert (raw(dw)[[0, 1, 1], [1, 0, 1]] == 0).all()


# ---- products over ragged groups -------------------------------------------------

def spread(rng, R, E, kind):
    if kind == "one":  # every row in one group, the others empty
        at = np.zeros(E + 1, np.int64)
        at[E // 2 + 1:] = R
        return at
    if kind == "behind":  # rows behind the last group
        return np.concatenate([[0], np.sort(rng.integers(0, max(1, R // 2) + 1, E))])
    return np.concatenate([[0], np.sort(rng.integers(0, R + 1, E - 1)), [R]])


CASES = [
    # dtype, rows, groups, N, K, spread, activation
    ("float32", 64, 4, 512, 512, "any", None), ("float32", 777, 13, 131, 65, "any", "gelu"),
    ("float32", 300, 3, 130, 260, "behind", "silu"), ("float32", 5, 9, 3, 1, "any", None),
    ("bfloat16", 1, 8, 264, 512, "any", "silu"), ("bfloat16", 16, 8, 1000, 1024, "any", "silu"),
    ("float16", 200, 5, 200, 72, "behind", None), ("bfloat16", 1024, 8, 640, 192, "any", "gelu"),
    ("float16", 777, 13, 283, 101, "any", "gelu"), ("bfloat16", 600, 2, 257, 129, "behind", "silu"),
    ("bfloat16", 500, 70, 72, 80, "any", None), ("float16", 2000, 1024, 40, 48, "any", None),
    ("bfloat16", 900, 7, 256, 384, "one", None), ("bfloat16", 1500, 4, 520, 1, "any", None),
    ("bfloat16", 1500, 2, 512, 256, "any", "gelu"), ("float16", 2100, 3, 700, 128, "behind", None),
    ("bfloat16", 40, 1, 96, 4104, "any", None), ("float16", 3, 3, 1, 1, "any", None),
    # few rows and a long sum, then 64 x 64 tiles, rows of four floats and others
    ("float32", 3, 1, 195, 5632, "any", None), ("float32", 70, 3, 260, 4099, "any", "gelu"),
    ("float32", 40, 9, 1027, 517, "behind", "silu"), ("float32", 1500, 3, 512, 640, "any", None),
    ("float32", 1500, 3, 515, 700, "behind", "silu"), ("float32", 2000, 2, 600, 70, "any", None),
]


@pytest.mark.parametrize("dtype,R,E,N,K,kind,act", CASES)
def test_grouped_linear(dtype, R, E, N, K, kind, act):
    g = cu()
    rng = np.random.default_rng(R + N)
    x, w = rnd(rng, (R, K), 1.0, dtype), rnd(rng, (E, N, K), K ** -0.5, dtype)
    b = rnd(rng, (E, N), 0.1, dtype)
    off = spread(rng, R, E, kind)
    xt, wt, ot, bt = up(x, dtype), up(w, dtype), ints(off), up(b, dtype)
    for bias, tb in ((None, None), (b, bt)):
        y, mag = ox.grouped_linear(x, w, off, bias)
        got = down(g.dev_grouped_linear(xt, wt, ot, tb))
        check_bound(got, y, gemm_bound(y, mag, K, dtype), "linear")
        assert (got[off[-1]:] == 0).all()
    if act:
        check_bound(down(g.dev_grouped_linear(xt, wt, ot, bt, act)), ox.act(y, act),
                    gemm_bound(ox.act(y, act), mag, K, dtype, act), act)
        assert (down(g.dev_grouped_linear(xt, wt, ot, bt, act))[off[-1]:] == 0).all()


@pytest.mark.parametrize("dtype,R,E,N,K,kind,act", CASES)
def test_grouped_linear_backward(dtype, R, E, N, K, kind, act):
    g = cu()
    rng = np.random.default_rng(R + N)
    x, w = rnd(rng, (R, K), 1.0, dtype), rnd(rng, (E, N, K), K ** -0.5, dtype)
    gr, pre = rnd(rng, (R, N), 1.0, dtype), rnd(rng, (R, N), 3.0, dtype)
    off = spread(rng, R, E, kind)
    # with an activation, grad act'(pre) is rounded to the operands' type: the
    # oracle takes that product as the device rounded it
    if act:
        through = g.empty((R, N), up(gr, dtype).dtype)
        lib = ctypes.CDLL(os.path.join(ROOT, "scaffolding_amd", "libsfgemm.so"))
        a, b = up(gr, dtype), up(pre, dtype)
        assert lib.sf_act_backward(P(a.data_ptr), P(b.data_ptr), P(through.data_ptr), I64(R * N), SFD[dtype],
                                   4 if act == "silu" else 5, None) == 0
        gg = down(through)
        want = gr.astype(np.float64) * ox.act_slope(pre, act)
        # half a step, and 16 fp32 steps of the slope's terms (at most 1.2 and,
        # for GELU, 2 x (c0 + 3 c1 x^2) s (1 - s) < 3)
        check_bound(gg, want, out_half_ulp_rel(dtype) * np.abs(want) + 16 * 4 * 2.0 ** -24 * np.abs(gr) + 2.0 ** -25,
                    "slope")
    else:
        gg = gr
    wants, mags = ox.grouped_linear_backward(gg, x, w, off)
    got = g.dev_grouped_linear_backward(up(gr, dtype), up(x, dtype), up(w, dtype), ints(off), True, act,
                                        up(pre, dtype) if act else None)
    for name, y, want, mag, n in zip(("dx", "dw", "db"), got, wants, mags, (N, R, R)):
        check_bound(down(y), want, gemm_bound(want, mag, n, dtype), name)
    assert (down(got[0])[off[-1]:] == 0).all()
    for e in range(E):
        if off[e] == off[e + 1]:
            assert (down(got[1])[e] == 0).all() and (down(got[2])[e] == 0).all()
    assert g.dev_grouped_linear_backward(up(gr, dtype), up(x, dtype), up(w, dtype), ints(off), False)[2] is None


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("R,E,N,K,kind,act", [(2000, 2, 1283, 1285, "any", "silu"), (2100, 3, 1285, 1283, "behind", None)])
def test_grouped_unaligned_128_tiles(dtype, R, E, N, K, kind, act):
    """Rows that start at any element, enough of them for 128 x 128 tiles."""
    test_grouped_linear(dtype, R, E, N, K, kind, act)
    test_grouped_linear_backward(dtype, R, E, N, K, kind, act)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("off", [[5, 30, 12, 99], [0, -7, 40, 20], [0, 0, 0, 0], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 0]])
def test_grouped_any_offsets(dtype, off):
    """Offsets that are not ascending from 0 within the rows: the ranges the
    documentation gives, nothing outside the operands."""
    g = cu()
    rng = np.random.default_rng(3)
    x, w, gr = rnd(rng, (50, 72), 1.0, dtype), rnd(rng, (3, 40, 72), 0.1, dtype), rnd(rng, (50, 40), 1.0, dtype)
    y, mag = ox.grouped_linear(x, w, off)
    check_bound(down(g.dev_grouped_linear(up(x, dtype), up(w, dtype), ints(off))), y, gemm_bound(y, mag, 72, dtype))
    wants, mags = ox.grouped_linear_backward(gr, x, w, off)
    got = g.dev_grouped_linear_backward(up(gr, dtype), up(x, dtype), up(w, dtype), ints(off))
    for a, want, m in zip(got, wants, mags):
        check_bound(down(a), want, gemm_bound(want, m, 72, dtype))


@pytest.mark.parametrize("dtype,R,N,K,ends", [
    # more 256 x 256 tiles than CUs: a short last round (in 128 x 128 tiles), a
    # long one, columns and rows that end inside a quarter, rows of no group
    ("bfloat16", 4096, 8192, 2048, [709, 1275, 1795, 2489, 2882, 3289, 3511, 4096]),
    ("float16", 4096, 8200, 2048, [10, 10, 2300, 4000]),
    ("bfloat16", 5000, 7000, 1920, [1, 1500, 1500, 2871, 4100]),
    ("bfloat16", 4100, 8192, 2048, [40 * i for i in range(1, 101)]),
])
def test_grouped_linear_many_tiles(dtype, R, N, K, ends):
    g = cu()
    rng = np.random.default_rng(R)
    E, off = len(ends), np.array([0] + ends)
    x = rnd(rng, (R, K), 1.0, dtype)
    # each group's weight: one matrix with its rows rotated
    base = rnd(rng, (N, K), K ** -0.5, dtype)
    w = np.stack([np.roll(base, e, 0) for e in range(E)]) if E < 10 else np.stack([base[:, ::(-1) ** e] for e in range(E)])
    b = rnd(rng, (E, N), 0.1, dtype)
    rows = np.unique(np.clip(np.concatenate([off[:-1], off[1:] - 1, off[:-1] + 127, off[:-1] + 128, off[:-1] + 256,
                                             rng.integers(0, R, 12), [R - 1]]), 0, R - 1))
    xt, wt, ot = up(x, dtype), up(w, dtype), ints(off)
    got = down(g.dev_grouped_linear(xt, wt, ot, up(b, dtype), "silu"))
    group = np.searchsorted(off[1:], rows, side="right")
    for r, e in zip(rows, group):
        if e == E:
            assert (got[r] == 0).all()
            continue
        y = x[r].astype(np.float64) @ w[e].astype(np.float64).T + b[e]
        mag = np.abs(x[r]).astype(np.float64) @ np.abs(w[e]).astype(np.float64).T
        check_bound(got[r], ox.act(y, "silu"), gemm_bound(ox.act(y, "silu"), mag, K, dtype, "silu"), "row %d" % r)
    assert (got[off[-1]:] == 0).all()
    # every row of the same group with the same input gives the same result
    same_rows = np.zeros((R, K), np.float32) + x[0]
    got = down(g.dev_grouped_linear(up(same_rows, dtype), wt, ot))
    for e in range(E):
        lo, hi = off[e], off[e + 1]
        assert (got[lo:hi] == got[lo:lo + 1]).all()


@pytest.mark.parametrize("dtype,R,N,K,ends", [
    ("bfloat16", 4096, 2048, 8192, [709, 1275, 1795, 2489, 2882, 3289, 3511, 4096]),
    ("float16", 3000, 2048, 8200, [0, 1100, 2900]),
])
def test_grouped_backward_many_tiles(dtype, R, N, K, ends):
    g = cu()
    rng = np.random.default_rng(R)
    E, off = len(ends), np.array([0] + ends)
    gr, x = rnd(rng, (R, N), 1.0, dtype), rnd(rng, (R, K), 1.0, dtype)
    base = rnd(rng, (N, K), N ** -0.5, dtype)
    w = np.stack([np.roll(base, e, 0) for e in range(E)])
    dx, dw, db = (down(t) for t in g.dev_grouped_linear_backward(up(gr, dtype), up(x, dtype), up(w, dtype), ints(off)))
    for r in np.unique(np.concatenate([off[off < R], off[1:] - 1, rng.integers(0, R, 8)])):
        if r < 0:
            continue
        e = int(np.searchsorted(off[1:], r, side="right"))
        if e == E:
            assert (dx[r] == 0).all()
            continue
        g64, w64 = gr[r].astype(np.float64), w[e].astype(np.float64)
        y, mag = g64 @ w64, np.abs(g64) @ np.abs(w64)
        check_bound(dx[r], y, gemm_bound(y, mag, N, dtype), "dx row %d" % r)
    for e in range(E):
        ge, xe = gr[off[e]:off[e + 1]].astype(np.float64), x[off[e]:off[e + 1]].astype(np.float64)
        for n in (0, 255, 256, N - 1, int(rng.integers(N))):
            y, mag = ge[:, n] @ xe, np.abs(ge[:, n]) @ np.abs(xe)
            check_bound(dw[e, n], y, gemm_bound(y, mag, max(1, len(ge)), dtype), "dw row %d" % n)
        s = ge.sum(0)
        check_bound(db[e], s, gemm_bound(s, np.abs(ge).sum(0), max(1, len(ge)), dtype), "db")


@pytest.mark.parametrize("R,E,N,K", [(0, 3, 8, 8), (8, 0, 8, 8), (8, 2, 0, 8), (8, 2, 8, 0)])
def test_grouped_empty(R, E, N, K):
    g = cu()
    z = [g.zeros(s, g.BFLOAT16) for s in ((R, K), (E, N, K), (E, N), (R, N))]
    off = ints(np.linspace(0, R, E + 1).astype(np.int32))
    y = down(g.dev_grouped_linear(z[0], z[1], off, z[2], "silu"))
    assert y.shape == (R, N) and (y == 0).all()
    dx, dw, db = g.dev_grouped_linear_backward(z[3], z[0], z[1], off)
    assert dx.shape == (R, K) and dw.shape == (E, N, K) and db.shape == (E, N)
    assert all((down(t) == 0).all() for t in (dx, dw, db))


def shifted(gt):
    """A copy of gt one element past the start of its memory: (memory, address)."""
    g = cu()
    size = np.dtype(gt.dtype).itemsize
    room = g.empty((gt.numel + 8,), gt.dtype)
    lib = ctypes.CDLL(os.path.join(ROOT, "scaffolding_amd", "libsfgemm.so"))
    assert lib.sf_memcpy_d2d(P(room.data_ptr + size), P(gt.data_ptr), ctypes.c_size_t(gt.nbytes), None) == 0
    return room, room.data_ptr + size


@pytest.mark.parametrize("dtype,R,E,N,K", [
    ("bfloat16", 30, 3, 72, 136), ("float16", 700, 2, 264, 256), ("float32", 90, 2, 68, 36), ("float32", 1500, 3, 512, 640),
    ("bfloat16", 9000, 2, 7168, 128),  # 256 x 256 tiles for aligned operands
])
@pytest.mark.parametrize("which", ["x", "w", "b", "y", "all"])
def test_grouped_operands_at_any_element(dtype, R, E, N, K, which):
    """Through the C ABI, each operand one element past an aligned address."""
    g = cu()
    rng = np.random.default_rng(R)
    x, w, b = rnd(rng, (R, K), 1.0, dtype), rnd(rng, (E, N, K), K ** -0.5, dtype), rnd(rng, (E, N), 1.0, dtype)
    off = np.array([R * i // (E + 1) for i in range(E + 1)])
    t = {"x": up(x, dtype), "w": up(w, dtype), "b": up(b, dtype)}
    t["y"] = g.zeros((R, N), t["x"].dtype)
    keep = {n: shifted(v) for n, v in t.items() if which in (n, "all")}
    at = {n: keep[n][1] if n in keep else v.data_ptr for n, v in t.items()}
    o = ints(off)
    lib = ctypes.CDLL(os.path.join(ROOT, "scaffolding_amd", "libsfgemm.so"))
    assert lib.sf_grouped_linear(P(at["x"]), P(at["w"]), P(o.data_ptr), P(at["b"]), P(at["y"]), I64(R), I64(E), I64(N),
                                 I64(K), SFD[dtype], 1, None) == 0
    back = g.empty((R, N), t["x"].dtype)
    assert lib.sf_memcpy_d2d(P(back.data_ptr), P(at["y"]), ctypes.c_size_t(back.nbytes), None) == 0
    got = down(back)
    rows = np.unique(np.concatenate([off[:-1], off[1:] - 1, rng.integers(0, off[-1], 60)]))
    e = np.searchsorted(off[1:], rows, side="right")
    for i in range(E):
        xe = x[rows[e == i]].astype(np.float64)
        y, mag = xe @ w[i].T.astype(np.float64) + b[i], np.abs(xe) @ np.abs(w[i]).T.astype(np.float64)
        check_bound(got[rows[e == i]], y, gemm_bound(y, mag + np.abs(b[i]), K, dtype))
    assert (got[off[-1]:] == 0).all()


def whole(rng, *shape):
    """Whole numbers of at most 3: every sum of their products is exact in
    fp32 up to 2^24 / 9 of them."""
    return rng.integers(-3, 4, shape, dtype=np.int8).astype(np.float32)


@pytest.mark.parametrize("N,K", [(2 ** 18 + 3, 1025), (1030, 2 ** 18 + 2)])
def test_fp32_weights_past_the_direct_loads(N, K):
    """One weight of more than 2^28 numbers: the register-staged tiles, and the
    small blocks for a few rows, forward and dX."""
    g = cu()
    rng = np.random.default_rng(N)
    w = whole(rng, 1, N, K)
    wt = f32(w)
    n, m = rng.integers(0, N, 40), rng.integers(0, K, 40)
    n[:3], m[:3] = (0, N - 1, N - 2), (0, K - 1, K - 2)
    for R, used in ((3, 3), (65, 61)):  # rows behind the only group too
        x, gr, off = whole(rng, R, K), whole(rng, R, N), ints([0, used])
        y = raw(g.dev_grouped_linear(f32(x), wt, off))
        assert np.array_equal(y[:used][:, n], x[:used].astype(np.float64) @ w[0][n].T.astype(np.float64))
        assert (y[used:] == 0).all()
        out = g.empty((R, K))
        a = f32(gr)
        lib = ctypes.CDLL(os.path.join(ROOT, "scaffolding_amd", "libsfgemm.so"))
        assert lib.sf_grouped_linear_dx(P(a.data_ptr), P(wt.data_ptr), P(off.data_ptr), P(out.data_ptr), I64(R), I64(1),
                                        I64(N), I64(K), 0, None) == 0
        dx = raw(out)
        assert np.array_equal(dx[:used][:, m], gr[:used].astype(np.float64) @ w[0][:, m].astype(np.float64))
        assert (dx[used:] == 0).all()


@pytest.mark.parametrize("N,K", [(2 ** 22 + 5, 3), (5, 2 ** 22 + 4)])
def test_fp32_weight_gradients_past_the_direct_loads(N, K):
    """Rows of so many numbers that all of them pass 2 GiB: dW by the
    register-staged tiles, an empty group and rows of none among them."""
    g = cu()
    rng = np.random.default_rng(N)
    R, off = 66, [0, 20, 20, 63]
    x, gr = whole(rng, R, K), whole(rng, R, N)
    a, b, o = f32(gr), f32(x), ints(off)
    dw, db = g.empty((3, N, K)), g.empty((3, N))
    lib = ctypes.CDLL(os.path.join(ROOT, "scaffolding_amd", "libsfgemm.so"))
    assert lib.sf_grouped_linear_dw(P(a.data_ptr), P(b.data_ptr), P(o.data_ptr), P(dw.data_ptr), P(db.data_ptr), I64(R),
                                    I64(3), I64(N), I64(K), 0, None) == 0
    dw, db = raw(dw), raw(db)
    for e in range(3):
        lo, hi = off[e], off[e + 1]
        assert np.array_equal(dw[e], gr[lo:hi].T @ x[lo:hi]) and np.array_equal(db[e], gr[lo:hi].sum(0))


def test_grouped_nan_stays_in_its_group():
    """A NaN of one group's rows, of rows of no group, or of an empty group's
    weight reaches no other output."""
    g = cu()
    rng = np.random.default_rng(5)
    x, w, gr = rnd(rng, (40, 64), 1.0, "bfloat16"), rnd(rng, (4, 64, 64), 0.1, "bfloat16"), rnd(rng, (40, 64), 1.0, "bfloat16")
    off = [0, 11, 11, 23, 30]
    x[11], gr[35], w[1] = np.nan, np.nan, np.nan
    x[38] = np.inf
    args = up(x, "bfloat16"), up(w, "bfloat16"), ints(off)
    y = down(g.dev_grouped_linear(*args))
    assert np.isnan(y[11]).all() and np.isfinite(np.delete(y, 11, 0)).all() and (y[30:] == 0).all()
    dx, dw, db = (down(t) for t in g.dev_grouped_linear_backward(up(gr, "bfloat16"), *args))
    assert np.isfinite(dx).all() and (dx[30:] == 0).all() and np.isfinite(db).all()
    assert np.isnan(dw[2]).all() and np.isfinite(dw[[0, 1, 3]]).all()


# ---- together ---------------------------------------------------------------------

def loss64(x, wr, w1, b1, w2, b2, g, e, off, slots, k):
    """The layer in fp64 for a given choice, and what its gradient needs."""
    T = x.shape[0]
    logits64 = x @ wr.T
    w = ox.route_weights(logits64, e)
    rows = np.zeros((T * k, x.shape[1]))
    rows[slots.reshape(-1)] = np.repeat(x, k, 0)
    pre = ox.grouped_linear(rows, w1, off, b1)[0]
    h = ox.act(pre, "silu")
    y = ox.grouped_linear(h, w2, off, b2)[0]
    out = (w[:, :, None] * y[slots]).sum(1)
    return (out * g).sum(), out, (logits64, w, rows, pre, h, y)


@pytest.mark.parametrize("T,E,k,D,H", [(1, 4, 2, 32, 48), (50, 6, 2, 64, 96), (200, 9, 3, 40, 72)])
def test_expert_layer_and_its_gradients(T, E, k, D, H):
    """Router, experts and combination forward and backward as a training step
    runs them, in fp32, against the fp64 formula and, for a few elements of
    each parameter, against its differences."""
    import scaffolding_amd as sf
    from scaffolding_amd.nn import functional as F

    rng = np.random.default_rng(T)
    shapes = dict(x=(T, D), wr=(E, D), w1=(E, H, D), b1=(E, H), w2=(E, D, H), b2=(E, D), g=(T, D))
    v = {n: (rng.standard_normal(s) * (0.3 if n[0] in "wb" else 1.0)).astype(np.float32) for n, s in shapes.items()}
    t = {n: sf.Tensor(a, device="cuda") for n, a in v.items()}
    lg = sf.matmul_nt(t["x"], t["wr"])
    r = F.route_topk(lg, k)
    rows = F.dispatch_rows(t["x"], r.slots)
    pre = F.grouped_linear(rows, t["w1"], r.offsets, t["b1"])
    h = F.grouped_linear(rows, t["w1"], r.offsets, t["b1"], "silu")
    y = F.grouped_linear(h, t["w2"], r.offsets, t["b2"])
    out = F.combine_rows(y, r.slots, r.weights)

    dy, dw = F.combine_rows_backward(t["g"], y, r.slots, r.weights)
    dh, dw2, db2 = F.grouped_linear_backward(dy, h, t["w2"], r.offsets)
    drows, dw1, db1 = F.grouped_linear_backward(dh, rows, t["w1"], r.offsets, True, "silu", pre)
    dl = F.route_topk_backward(dw, lg, r)
    dx = F.combine_rows(drows, r.slots).numpy() + sf.matmul(dl, t["wr"]).numpy()
    dwr = dl.numpy().astype(np.float64).T @ v["x"]

    e, off, slots = r.experts.numpy(), r.offsets.numpy(), r.slots.numpy()
    m = {n: a.astype(np.float64) for n, a in v.items()}
    val, out64, (lg64, w64, rows64, pre64, h64, y64) = loss64(**m, e=e, off=off, slots=slots, k=k)
    assert np.array_equal(e, ox.route(lg.numpy(), k)[1])
    dy64 = np.zeros((T * k, D))
    for j in range(k):
        dy64[slots[:, j]] = w64[:, j, None] * m["g"]
    dww = (m["g"][:, None] * y64[slots]).sum(2)
    (dh64, dw2_64, db2_64), _ = ox.grouped_linear_backward(dy64, h64, m["w2"], off)
    (dr64, dw1_64, db1_64), _ = ox.grouped_linear_backward(dh64 * ox.act_slope(pre64, "silu"), rows64, m["w1"], off)
    dl64 = ox.route_backward(dww, lg64, e)
    want = dict(x=dr64[slots].sum(1) + dl64 @ m["wr"], wr=dl64.T @ m["x"], w1=dw1_64, b1=db1_64, w2=dw2_64, b2=db2_64)
    got = dict(x=dx, wr=dwr, w1=dw1.numpy(), b1=db1.numpy(), w2=dw2.numpy(), b2=db2.numpy())
    # chains of fp32 sums of at most T k + D + H terms: normwise 2^-24 per
    # term and stage, six stages
    tol = 6 * (T * k + D + H) * 2.0 ** -24

    def near(a, b):
        return np.linalg.norm(a - b) <= tol * max(np.linalg.norm(b), 1e-3)

    assert near(out.numpy(), out64)
    for n in want:
        assert near(got[n], want[n]), n
        flat = want[n].reshape(-1)
        for i in rng.choice(flat.size, 4):
            step = 1e-6
            hi, lo = dict(m), dict(m)
            hi[n], lo[n] = m[n].copy(), m[n].copy()
            hi[n].reshape(-1)[i] += step
            lo[n].reshape(-1)[i] -= step
            num = (loss64(**hi, e=e, off=off, slots=slots, k=k)[0] - loss64(**lo, e=e, off=off, slots=slots, k=k)[0]) / (2 * step)
            assert abs(num - flat[i]) <= 1e-5 * max(1.0, abs(flat[i])), n


# ---- streams, graphs, devices -------------------------------------------------------

class Chain:
    """Routing, dispatch, a grouped product with its gradients and combination
    through the C entries, all buffers fixed, on a given stream."""

    def __init__(self, seed, T=200, E=6, k=2, D=128, H=192, dtype="bfloat16"):
        g = cu()
        rng = np.random.default_rng(seed)
        self.lib = ctypes.CDLL(os.path.join(ROOT, "scaffolding_amd", "libsfgemm.so"))
        self.lib.sf_route_topk_work.restype = I64
        dt = up(np.zeros(1), dtype).dtype
        self.n = dict(T=T, E=E, k=k, D=D, H=H, dt=SFD[dtype])
        self.x, self.lg = up(rnd(rng, (T, D), 1.0, dtype), dtype), up(rnd(rng, (T, E), 1.0, dtype), dtype)
        self.w = up(rnd(rng, (E, H, D), 0.1, dtype), dtype)
        i32 = np.dtype(np.int32)
        self.out = dict(wt=g.empty((T, k)), ex=g.empty((T, k), i32), off=g.empty((E + 1,), i32),
                        sl=g.empty((T, k), i32), rows=g.empty((T * k, D), dt), y=g.empty((T * k, H), dt),
                        z=g.empty((T, H), dt), dx=g.empty((T * k, D), dt), dw=g.empty((E, H, D), dt),
                        db=g.empty((E, H), dt), dr=g.empty((T * k, H), dt), dwt=g.empty((T, k)),
                        dl=g.empty((T, E), dt))
        self.work = g.empty((max(1, self.lib.sf_route_topk_work(I64(T), I64(E)) // 4),), i32)

    def run(self, st):
        lib, n, o = self.lib, self.n, {a: P(t.data_ptr) for a, t in self.out.items()}
        T, E, k, D, H, dt = I64(n["T"]), I64(n["E"]), I64(n["k"]), I64(n["D"]), I64(n["H"]), n["dt"]
        R = I64(n["T"] * n["k"])
        x, lg, w = P(self.x.data_ptr), P(self.lg.data_ptr), P(self.w.data_ptr)
        rcs = [lib.sf_route_topk(lg, T, E, k, dt, 1, o["wt"], o["ex"], o["off"], o["sl"], P(self.work.data_ptr), st),
               lib.sf_dispatch_rows(x, o["sl"], o["rows"], T, k, D, dt, st),
               lib.sf_grouped_linear(o["rows"], w, o["off"], None, o["y"], R, E, H, D, dt, 4, st),
               lib.sf_combine_rows(o["y"], o["sl"], o["wt"], o["z"], T, k, H, dt, st),
               lib.sf_combine_rows_backward(o["z"], o["y"], o["sl"], o["wt"], o["dr"], o["dwt"], T, k, H, dt, st),
               lib.sf_grouped_linear_dx(o["dr"], w, o["off"], o["dx"], R, E, H, D, dt, st),
               lib.sf_grouped_linear_dw(o["dr"], o["rows"], o["off"], o["dw"], o["db"], R, E, H, D, dt, st),
               lib.sf_route_topk_backward(o["dwt"], lg, o["wt"], o["ex"], T, E, k, dt, 1, o["dl"], st)]
        assert rcs == [0] * len(rcs), rcs

    def clear(self, st=None):
        for t in self.out.values():
            assert self.lib.sf_zero(P(t.data_ptr), ctypes.c_size_t(t.nbytes), st) == 0

    def values(self):
        return {n: down(t) if t.dtype != np.int32 else raw(t) for n, t in self.out.items()}


def same(a, b):
    assert all(np.array_equal(a[n], b[n]) for n in a), [n for n in a if not np.array_equal(a[n], b[n])]


def test_two_streams_and_repeated_calls():
    g = cu()
    a, b = Chain(1), Chain(2, T=333, E=11)
    a.run(None)
    b.run(None)
    wa, wb = a.values(), b.values()
    a.run(None)
    same(a.values(), wa)  # the same bits again
    st = [P(), P()]
    for s in st:
        assert a.lib.sf_stream_create(ctypes.byref(s)) == 0
    a.clear()
    b.clear()
    g.device_synchronize()
    for _ in range(3):
        a.run(st[0])
        b.run(st[1])
    for s in st:
        assert a.lib.sf_stream_synchronize(s) == 0
        a.lib.sf_stream_destroy(s)
    same(a.values(), wa)
    same(b.values(), wb)


def test_two_captured_graphs():
    """Two graphs of the whole chain, replayed in turn with eager calls and
    synchronisations between: every replay gives the eager bits."""
    g = cu()
    hip = ctypes.CDLL("libamdhip64.so.7")
    chains = [Chain(1), Chain(2, T=500, E=3)]
    want, graphs = [], []
    for c in chains:
        c.run(None)
        want.append(c.values())
    st = P()
    lib = chains[0].lib
    assert lib.sf_stream_create(ctypes.byref(st)) == 0
    for c in chains:
        graph, ex = P(), P()
        assert hip.hipStreamBeginCapture(st, 0) == 0
        c.run(st)
        assert hip.hipStreamEndCapture(st, ctypes.byref(graph)) == 0
        assert hip.hipGraphInstantiate(ctypes.byref(ex), graph, None, None, ctypes.c_size_t(0)) == 0
        graphs.append((graph, ex))
    for i in range(3):
        Chain(5 + i).run(None)
        g.device_synchronize()
        for c, (_, ex), w in zip(chains, graphs, want):
            c.clear(st)
            assert hip.hipGraphLaunch(ex, st) == 0
        assert lib.sf_stream_synchronize(st) == 0
        for c, w in zip(chains, want):
            same(c.values(), w)
    for graph, ex in graphs:
        hip.hipGraphExecDestroy(ex)
        hip.hipGraphDestroy(graph)
    lib.sf_stream_destroy(st)


def test_a_long_operand():
    """Rows past 2^31 elements: 64-bit row offsets in every kernel."""
    g = cu()
    R, C = 70000, 32768  # 2.3e9 elements of 2 bytes
    x = g.zeros((R, C), g.BFLOAT16)
    rng = np.random.default_rng(0)
    last = rnd(rng, (8, C), 1.0, "bfloat16")
    lib = ctypes.CDLL(os.path.join(ROOT, "scaffolding_amd", "libsfgemm.so"))
    tail = up(last, "bfloat16")
    assert lib.sf_memcpy_d2d(P(x.data_ptr + (R - 8) * C * 2), P(tail.data_ptr), ctypes.c_size_t(8 * C * 2), None) == 0
    w = rnd(rng, (2, 16, C), C ** -0.5, "bfloat16")
    off = [0, R - 5, R]
    y = down(g.dev_grouped_linear(x, up(w, "bfloat16"), ints(off)))
    want, mag = ox.grouped_linear(last, w, [0, 3, 8])
    check_bound(y[-8:], want, gemm_bound(want, mag, C, "bfloat16"))
    assert (y[:-8] == 0).all()
    gr = np.zeros((R, 16), np.float32)
    gr[-8:] = rnd(rng, (8, 16), 1.0, "bfloat16")
    _, dw, _ = g.dev_grouped_linear_backward(up(gr, "bfloat16"), x, up(w, "bfloat16"), ints(off), False)
    (_, want, _), (_, mag, _) = ox.grouped_linear_backward(gr[-8:], last, w, [0, 3, 8])
    check_bound(down(dw), want, gemm_bound(want, mag, 8, "bfloat16"))
    slots = np.arange(R).reshape(R // 2, 2)[:, ::-1]
    z = g.dev_combine_rows(x, ints(slots))
    got = np.empty((4, C), np.uint16)
    assert lib.sf_memcpy_d2h(got.ctypes.data_as(P), P(z.data_ptr + (R // 2 - 4) * C * 2), ctypes.c_size_t(4 * C * 2),
                             None) == 0
    pair = last.reshape(4, 2, C).astype(np.float64).sum(1)
    check_bound((got.astype(np.uint32) << 16).view(np.float32), pair, 2.0 ** -8 * np.abs(pair) + 1e-30)


def test_fp32_gradient_of_a_very_wide_layer_with_few_outputs():
    """The direct loads step through 64 rows of the weight at a time: with so
    few outputs that those reach past 4 GiB from its start, an infinite weight
    must still meet only its own product."""
    g = cu()
    N, K = 7, 2 ** 25
    w = g.zeros((1, N, K), np.float32)
    lib = ctypes.CDLL(os.path.join(ROOT, "scaffolding_amd", "libsfgemm.so"))
    block = np.zeros((N, 8), np.float32)
    block[0, 5], block[3, 1], block[6, 2] = np.inf, 2.0, -3.0
    for n in range(N):
        row = np.ascontiguousarray(block[n])
        assert lib.sf_memcpy_h2d(P(w.data_ptr + n * K * 4), row.ctypes.data_as(P), ctypes.c_size_t(32), None) == 0
    for R in (1, 70):
        out = g.empty((R, K))
        a, o = f32(np.ones((R, N))), ints([0, R])
        assert lib.sf_grouped_linear_dx(P(a.data_ptr), P(w.data_ptr), P(o.data_ptr), P(out.data_ptr), I64(R), I64(1),
                                        I64(N), I64(K), 0, None) == 0
        for r in (0, R - 1):
            got = np.empty(K if r == 0 else 4096, np.float32)
            assert lib.sf_memcpy_d2h(got.ctypes.data_as(P), P(out.data_ptr + r * K * 4), ctypes.c_size_t(got.nbytes),
                                     None) == 0
            assert got[:8].tolist() == [0, 2, -3, 0, 0, np.inf, 0, 0] and (got[8:] == 0).all()

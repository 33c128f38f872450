"""Expert operators without a GPU: the oracle against itself (gradients
against differences), and every refusal of the C entries and the seam, which
are all made before the device is touched."""
from __future__ import annotations

import ctypes
import os

import numpy as np
import pytest

from oracle import experts as ox

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
I64, P = ctypes.c_int64, ctypes.c_void_p
A = P(4096)  # never dereferenced


@pytest.fixture(scope="module")
def lib():
    so = ctypes.CDLL(os.path.join(ROOT, "scaffolding_amd", "libsfgemm.so"))
    so.sf_last_error.restype = ctypes.c_char_p
    so.sf_route_topk_work.restype = I64
    return so


# ---- the oracle -----------------------------------------------------------

def test_oracle_routing_by_hand():
    inf, nan = np.inf, np.nan
    w, e, off, slots = ox.route([[1.0, 3.0, 3.0], [-inf, -inf, -inf], [0.0, nan, 5.0]], 2)
    assert e.tolist() == [[1, 2], [0, 1], [1, 2]]
    assert w[0].tolist() == [0.5, 0.5] and w[1].tolist() == [0.0, 0.0] and np.isnan(w[2]).all()
    assert off.tolist() == [0, 1, 4, 6] and slots.tolist() == [[1, 4], [0, 2], [3, 5]]


@pytest.mark.parametrize("renorm", [True, False])
def test_oracle_routing_gradient_against_differences(renorm):
    rng = np.random.default_rng(0)
    v, g = rng.standard_normal((5, 7)), rng.standard_normal((5, 3))
    _, e, _, _ = ox.route(v, 3)
    d = ox.route_backward(g, v, e, renorm)
    h = 1e-6
    for t in range(5):
        for j in range(7):
            a, b = v.copy(), v.copy()
            a[t, j] += h
            b[t, j] -= h
            num = ((ox.route_weights(a, e, renorm) - ox.route_weights(b, e, renorm)) * g).sum() / (2 * h)
            assert abs(num - d[t, j]) < 1e-8


def test_oracle_grouped_gradients_against_differences():
    rng = np.random.default_rng(1)
    x, w, g = rng.standard_normal((6, 4)), rng.standard_normal((3, 5, 4)), rng.standard_normal((6, 5))
    off = [0, 2, 2, 5]  # an empty group, a row behind the last

    def loss(x, w):
        return (ox.act(ox.grouped_linear(x, w, off)[0], "silu") * g).sum()

    y, _ = ox.grouped_linear(x, w, off)
    assert (y[5] == 0).all()
    (dx, dw, db), _ = ox.grouped_linear_backward(g * ox.act_slope(y, "silu"), x, w, off)
    h = 1e-6
    for i in np.ndindex(x.shape):
        a, b = x.copy(), x.copy()
        a[i] += h
        b[i] -= h
        assert abs((loss(a, w) - loss(b, w)) / (2 * h) - dx[i]) < 1e-7
    for i in np.ndindex(w.shape):
        a, b = w.copy(), w.copy()
        a[i] += h
        b[i] -= h
        assert abs((loss(x, a) - loss(x, b)) / (2 * h) - dw[i]) < 1e-7


@pytest.mark.parametrize("name", ["silu", "gelu"])
def test_oracle_activation_slopes(name):
    v = np.linspace(-6, 6, 101)
    num = (ox.act(v + 1e-6, name) - ox.act(v - 1e-6, name)) / 2e-6
    assert np.max(np.abs(num - ox.act_slope(v, name))) < 1e-8


@pytest.mark.parametrize("offsets,rows,want", [
    ([0, 3, 3, 8], 10, [(0, 3), (3, 3), (3, 8)]),
    ([5, 3, 1, 20], 10, [(0, 3), (3, 3), (3, 10)]),
    ([0, -4, 7, 2], 10, [(0, 0), (0, 7), (7, 7)]),
])
def test_oracle_group_ranges(offsets, rows, want):
    assert ox.groups(offsets, rows) == want


# ---- refusals of the C entries ------------------------------------------------

def route(lib, T=4, E=8, k=2, dt=0, logits=A, w=A, e=A, o=A, s=A, work=A):
    return lib.sf_route_topk(logits, I64(T), I64(E), I64(k), dt, 1, w, e, o, s, work, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dt=7), -2, b"dtype"), (dict(T=-1), -2, b"tokens"), (dict(E=0), -2, b"experts"), (dict(k=0), -2, b"k"),
    (dict(k=9), -2, b"k"), (dict(E=1025), -3, b"experts"), (dict(E=40, k=17), -3, b"k"),
    (dict(T=2 ** 31 - 1), -3, b"2^31"), (dict(T=2 ** 30, k=2), -3, b"2^31"), (dict(T=2 ** 26, k=1), -3, b"2^26"),
    (dict(logits=None), -2, b"null"), (dict(w=None), -2, b"null"), (dict(e=None), -2, b"null"),
    (dict(o=None), -2, b"null"), (dict(s=None), -2, b"null"), (dict(T=65, work=None), -2, b"null"),
])
def test_route_refusals(lib, kw, code, text):
    assert route(lib, **kw) == code
    assert text in lib.sf_last_error()


def test_route_work(lib):
    assert lib.sf_route_topk_work(I64(0), I64(8)) == 0
    assert lib.sf_route_topk_work(I64(64), I64(8)) == 0
    assert lib.sf_route_topk_work(I64(65), I64(8)) == 3 * 8 * 4


@pytest.mark.parametrize("kw,code", [
    (dict(dt=-1), -2), (dict(k=5, E=4), -2), (dict(E=1025), -3), (dict(g=None), -2), (dict(out=None), -2),
    (dict(T=2 ** 26), -3),
])
def test_route_backward_refusals(lib, kw, code):
    d = dict(T=4, E=8, k=2, dt=0, g=A, out=A)
    d.update(kw)
    assert lib.sf_route_topk_backward(d["g"], A, A, A, I64(d["T"]), I64(d["E"]), I64(d["k"]), d["dt"], 1, d["out"],
                                      None) == code
    assert lib.sf_last_error() != b""


@pytest.mark.parametrize("kw,code", [
    (dict(dt=9), -2), (dict(T=-1), -2), (dict(k=0), -2), (dict(D=-1), -2), (dict(T=2 ** 30, k=2), -3),
    (dict(T=2 ** 40, k=2 ** 40), -3), (dict(D=2 ** 31), -3), (dict(D=2 ** 30 + 1), -3),
    (dict(T=2 ** 26, k=1, D=2048), -3), (dict(a=None), -2), (dict(s=None), -2),
    (dict(out=None), -2),
])
def test_row_exchange_refusals(lib, kw, code):
    d = dict(T=4, k=2, D=8, dt=0, a=A, s=A, out=A)
    d.update(kw)
    size = (I64(d["T"]), I64(d["k"]), I64(d["D"]), d["dt"], None)
    assert lib.sf_dispatch_rows(d["a"], d["s"], d["out"], *size) == code
    assert lib.sf_combine_rows(d["a"], d["s"], A, d["out"], *size) == code
    assert lib.sf_combine_rows_backward(d["a"], A, d["s"], A, d["out"], A, *size) == code
    assert lib.sf_last_error() != b""


def test_row_exchange_empty(lib):
    for T, D in ((0, 8), (4, 0)):
        size = (I64(T), I64(2), I64(D), 0, None)
        assert lib.sf_dispatch_rows(None, None, None, *size) == 0
        assert lib.sf_combine_rows(None, None, None, None, *size) == 0
    assert lib.sf_combine_rows_backward(None, None, None, None, None, None, I64(0), I64(2), I64(8), 0, None) == 0


@pytest.mark.parametrize("kw,code,text", [
    (dict(dt=3), -2, b"dtype"), (dict(R=-1), -2, b"negative"), (dict(E=-1), -2, b"negative"),
    (dict(N=-1), -2, b"negative"), (dict(K=-1), -2, b"negative"), (dict(E=1025), -3, b"groups"),
    (dict(R=2 ** 31), -3, b"2^31"), (dict(N=2 ** 31), -3, b"2^31"), (dict(K=2 ** 31), -3, b"2^31"),
    (dict(R=2 ** 30 + 1), -3, b"2^30"), (dict(N=2 ** 30 + 1), -3, b"2^30"), (dict(K=2 ** 30 + 1), -3, b"2^30"),
    (dict(a=None), -2, b"null"), (dict(b=None), -2, b"null"), (dict(o=None), -2, b"null"),
    (dict(out=None), -2, b"null"),
])
def test_grouped_refusals(lib, kw, code, text):
    d = dict(R=8, E=2, N=16, K=16, dt=2, a=A, b=A, o=A, out=A)
    d.update(kw)
    size = (I64(d["R"]), I64(d["E"]), I64(d["N"]), I64(d["K"]), d["dt"])
    for rc in (lib.sf_grouped_linear(d["a"], d["b"], d["o"], None, d["out"], *size, 0, None),
               lib.sf_grouped_linear_dx(d["a"], d["b"], d["o"], d["out"], *size, None),
               lib.sf_grouped_linear_dw(d["a"], d["b"], d["o"], d["out"], None, *size, None)):
        assert rc == code
        assert text in lib.sf_last_error()


def test_grouped_refusals_of_one_entry(lib):
    assert lib.sf_grouped_linear_dw(A, None, A, None, A, I64(8), I64(2), I64(2 ** 28 + 1), I64(0), 2, None) == -3
    assert b"2^28" in lib.sf_last_error()
    size = (I64(8), I64(2), I64(16), I64(16), 2)
    assert lib.sf_grouped_linear(A, A, A, None, A, *size, 6, None) == -2
    assert b"epilogue" in lib.sf_last_error()
    assert lib.sf_grouped_linear(A, A, A, None, A, *size, 1, None) == -2
    assert b"bias" in lib.sf_last_error()
    # a grid past 2^22 tiles
    assert lib.sf_grouped_linear(A, A, A, None, A, I64(2 ** 22), I64(4), I64(2 ** 16), I64(8), 2, 0, None) == -3
    assert lib.sf_grouped_linear_dw(A, A, A, A, None, I64(8), I64(1024), I64(2 ** 16), I64(2 ** 16), 2, None) == -3
    assert lib.sf_act_backward(A, A, A, I64(8), 2, 0, None) == -2
    assert lib.sf_act_backward(A, A, A, I64(-1), 2, 4, None) == -2
    assert lib.sf_act_backward(A, A, A, I64(8), 5, 4, None) == -2
    assert lib.sf_act_backward(A, None, A, I64(8), 2, 4, None) == -2
    assert lib.sf_act_backward(None, None, None, I64(0), 2, 4, None) == 0


def test_grouped_empty(lib):
    def size(R, E, N, K):
        return I64(R), I64(E), I64(N), I64(K), 2

    assert lib.sf_grouped_linear(None, None, None, None, None, *size(0, 2, 16, 16), 0, None) == 0
    assert lib.sf_grouped_linear(None, None, None, None, None, *size(8, 2, 0, 16), 0, None) == 0
    assert lib.sf_grouped_linear_dx(None, None, None, None, *size(8, 2, 16, 0), None) == 0
    assert lib.sf_grouped_linear_dw(None, None, None, None, None, *size(8, 0, 16, 16), None) == 0


# ---- refusals of the seam -------------------------------------------------------

def fake(shape, dtype="float32", dev=0):
    """A tensor without memory: the seam's checks read only its description."""
    from scaffolding_amd import _cuda_ops as g
    return g.GpuTensor(g.CudaBuffer(), tuple(shape), g.resolve_dtype(dtype), dev)


def raises(exc, f, *a):
    with pytest.raises(exc):
        f(*a)


def test_seam_refusals():
    from scaffolding_amd import _cuda_ops as g
    f, i = fake, lambda *s: fake(s, "int32")
    raises(ValueError, g.dev_route_topk, f((4, 8)), 9)
    raises(ValueError, g.dev_route_topk, f((4, 8)), 0)
    raises(ValueError, g.dev_route_topk, f(()), 1)
    raises(TypeError, g.dev_route_topk, i(4, 8), 2)
    raises(TypeError, g.dev_route_topk_backward, f((4, 2), "float16"), f((4, 8)), f((4, 2)), i(4, 2))
    raises(TypeError, g.dev_route_topk_backward, f((4, 2)), f((4, 8)), f((4, 2)), f((4, 2)))
    raises(ValueError, g.dev_route_topk_backward, f((4, 3)), f((4, 8)), f((4, 2)), i(4, 2))
    raises(ValueError, g.dev_route_topk_backward, f((3, 2)), f((4, 8)), f((3, 2)), i(3, 2))
    raises(ValueError, g.dev_dispatch_rows, f((4, 8)), i(3, 2))
    raises(ValueError, g.dev_dispatch_rows, f((4, 8)), i(4))
    raises(TypeError, g.dev_dispatch_rows, f((4, 8)), f((4, 2)))
    raises(TypeError, g.dev_dispatch_rows, i(4, 8), i(4, 2))
    raises(ValueError, g.dev_dispatch_rows, f((4, 8)), fake((4, 2), "int32", 1))
    raises(ValueError, g.dev_combine_rows, f((7, 8)), i(4, 2))
    raises(ValueError, g.dev_combine_rows, f((8, 8)), i(4, 2), f((4, 3)))
    raises(TypeError, g.dev_combine_rows, f((8, 8)), i(4, 2), f((4, 2), "bfloat16"))
    raises(ValueError, g.dev_combine_rows_backward, f((4, 7)), f((8, 8)), i(4, 2), f((4, 2)))
    raises(TypeError, g.dev_combine_rows_backward, f((4, 8), "float16"), f((8, 8)), i(4, 2), f((4, 2)))
    x, w, o = f((8, 16)), f((2, 4, 16)), i(3)
    raises(ValueError, g.dev_grouped_linear, f((8, 15)), w, o)
    raises(ValueError, g.dev_grouped_linear, f((2, 4, 16)), w, o)
    raises(ValueError, g.dev_grouped_linear, x, f((4, 16)), o)
    raises(ValueError, g.dev_grouped_linear, x, w, i(2))
    raises(TypeError, g.dev_grouped_linear, x, w, f((3,)))
    raises(TypeError, g.dev_grouped_linear, x, f((2, 4, 16), "float16"), o)
    raises(ValueError, g.dev_grouped_linear, x, w, o, f((4,)))
    raises(TypeError, g.dev_grouped_linear, x, w, o, f((2, 4), "float16"))
    raises(ValueError, g.dev_grouped_linear, x, w, o, None, "relu")
    raises(ValueError, g.dev_grouped_linear, x, fake((2, 4, 16), dev=1), o)
    gr = f((8, 4))
    raises(ValueError, g.dev_grouped_linear_backward, f((8, 5)), x, w, o)
    raises(ValueError, g.dev_grouped_linear_backward, gr, f((7, 16)), w, o)
    raises(ValueError, g.dev_grouped_linear_backward, gr, x, w, o, True, "silu")
    raises(ValueError, g.dev_grouped_linear_backward, gr, x, w, o, True, "silu", f((8, 5)))
    raises(TypeError, g.dev_grouped_linear_backward, gr, x, w, o, True, "silu", f((8, 4), "float16"))
    raises(ValueError, g.dev_grouped_linear_backward, gr, x, w, o, True, "tanh")


def test_cpu_tensors_are_refused():
    import scaffolding_amd as sf
    from scaffolding_amd.nn import functional as F
    t = sf.Tensor(np.zeros((4, 8), np.float32))
    raises(RuntimeError, F.route_topk, t, 2)
    raises(RuntimeError, F.grouped_linear, t, t, t)
    raises(RuntimeError, F.dispatch_rows, t, t)
    raises(RuntimeError, F.combine_rows, t, t)


def test_integer_tensors_on_the_host():
    import scaffolding_amd as sf
    t = sf.Tensor(np.array([1, 2]), dtype="int32")
    assert t.dtype is sf.int32 and t.dtype.itemsize == 4 and t.numpy().dtype == np.int32
    assert sf.uint8.itemsize == 1
    # without a dtype, integers become float32 as before
    assert sf.Tensor(np.array([1, 2], np.int32)).dtype is sf.float32


@pytest.mark.parametrize("T", [2 ** 26 - 3, 2 ** 26 - 1])
def test_routing_refuses_grids_past_the_launch_limit(lib, T):
    """The gradient takes 64 threads a token in blocks of four tokens: 2^26 - 4
    tokens are the last whose grid stays below 2^32 threads."""
    assert -(-T // 4) * 256 >= 2 ** 32 > -(-(2 ** 26 - 4) // 4) * 256
    assert route(lib, T=T, k=1) == -3 and b"2^26" in lib.sf_last_error()
    assert lib.sf_route_topk_backward(A, A, A, A, I64(T), I64(8), I64(1), 0, 1, A, None) == -3
    assert b"2^26" in lib.sf_last_error()

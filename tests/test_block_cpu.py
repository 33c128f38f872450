"""Operators of a causal transformer block without a GPU: the oracle against
itself (gradients against differences), and every refusal of the C entries and
the seam, which are all made before the device is touched."""
from __future__ import annotations

import ctypes
import os

import numpy as np
import pytest

from oracle import block as ox

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
I64, P, F32 = ctypes.c_int64, ctypes.c_void_p, ctypes.c_float
A = P(4096)  # never dereferenced
INVALID, UNSUPPORTED = -2, -3


@pytest.fixture(scope="module")
def lib():
    so = ctypes.CDLL(os.path.join(ROOT, "scaffolding_amd", "libsfgemm.so"))
    so.sf_last_error.restype = ctypes.c_char_p
    for name in ("sf_qk_norm_rope_backward_work", "sf_window_attention_backward_work",
                 "sf_window_attention_cached_work", "sf_gated_backward_work"):
        getattr(so, name).restype = I64
    return so


def call(f, *args):
    """Integers as int64 but for those wrapped already."""
    return f(*[I64(a) if type(a) is int else a for a in args])


def c_int(v):
    return ctypes.c_int(v)


# ---- the oracle -----------------------------------------------------------

def differences(loss, x, grad, h=1e-6, tol=2e-8):
    """Central differences of a loss of size ~1 and second derivatives of size
    ~10: rounding 2^-53 / h and truncation h^2 stay below 1e-9."""
    for i in np.ndindex(x.shape):
        a, b = x.copy(), x.copy()
        a[i] += h
        b[i] -= h
        assert abs((loss(a) - loss(b)) / (2 * h) - grad[i]) < tol * max(1.0, np.abs(grad).max())


def test_oracle_rotation_by_hand():
    t = ox.rope_table(4, 2)
    x = np.zeros((1, 2, 1, 3))
    x[0, :, 0] = [1.0, 0.0, 5.0]
    y = ox.rotate(x, t, np.array([[0, 3]]), False)
    assert np.allclose(y[0, 0, 0], [1, 0, 5]) and np.allclose(y[0, 1, 0], [np.cos(3), np.sin(3), 5])
    assert np.isnan(ox.rotate(x, t, np.array([[4, -1]]), True)[0, :, 0, :2]).all()
    assert ox.pairs_of(4, False) == [(0, 2), (1, 3)] and ox.pairs_of(4, True) == [(0, 1), (2, 3)]


@pytest.mark.parametrize("kind,interleaved", [("rms", False), ("layer", True)])
def test_oracle_norm_rope_gradients_against_differences(kind, interleaved):
    rng = np.random.default_rng(0)
    H, Hk, D = 2, 1, 6
    x, g = (rng.standard_normal((1, 3, (H + 2 * Hk) * D)) for _ in range(2))
    w, b = rng.standard_normal((2, D)), rng.standard_normal((2, D))
    t, pos = ox.rope_table(9, 4), np.array([[0, 8, 3]])

    def loss(x=x, w=w, b=b):
        return (ox.qk_norm_rope(x, H, Hk, t, pos, w, b, kind, 1e-3, interleaved)[0] * g).sum()

    (dx, dw, db), _ = ox.qk_norm_rope_backward(g, x, H, Hk, t, pos, w, kind, 1e-3, interleaved)
    differences(lambda v: loss(x=v), x, dx)
    differences(lambda v: loss(w=v), w, dw)
    differences(lambda v: loss(b=v), b, db)


@pytest.mark.parametrize("window,sinks,lengths", [(None, 0, None), (2, 1, None), (3, 0, [4, 0]), (1, 2, [9, 5])])
def test_oracle_window_gradients_against_differences(window, sinks, lengths):
    rng = np.random.default_rng(1)
    H, Hk, D, N = 4, 2, 2, 6
    x, g = rng.standard_normal((2, N, (H + 2 * Hk) * D)), rng.standard_normal((2, N, H * D))

    def loss(v):
        return (ox.window_attention(v, H, Hk, window, sinks, 0.7, lengths)[0] * g).sum()

    differences(loss, x, ox.window_attention_backward(g, x, H, Hk, window, sinks, 0.7, lengths)[0])


def test_oracle_window_over_a_cache_is_the_whole_sequence():
    rng = np.random.default_rng(2)
    H, Hk, D, N = 4, 2, 3, 9
    x = rng.standard_normal((2, N, (H + 2 * Hk) * D))
    want, _ = ox.window_attention(x, H, Hk, 4, 1, 0.5)
    q, k, v = (a.reshape(2, N, -1) for a in ox.split_heads(x, H, Hk))
    got = ox.window_attention_cached(q[:, 5:8], k, v, [5, 5], H, Hk, 4, 1, 0.5)
    assert np.abs(got - want[:, 5:8]).max() < 1e-12


@pytest.mark.parametrize("kind", [None, "silu", "gelu"])
def test_oracle_gated_gradients_against_differences(kind):
    rng = np.random.default_rng(3)
    x, W, b, g = (rng.standard_normal(s) for s in ((4, 3), (10, 3), (10,), (4, 5)))

    def loss(x=x, W=W, b=b):
        return (ox.gated(x, W, b, kind)[0] * g).sum()

    dx, dW, db, dpre = ox.gated_backward(g, x, W, ox.gated(x, W, b, kind)[1], kind)
    differences(lambda v: loss(x=v), x, dx)
    differences(lambda v: loss(W=v), W, dW)
    differences(lambda v: loss(b=v), b, db)
    assert np.allclose(dpre.sum(0), db)


# ---- refusals of the C entries ------------------------------------------------

def norm_rope(lib, **kw):
    d = dict(x=A, ldx=64, q=A, k=A, v=A, ldq=32, ldk=16, ldv=16, s=128, table=A, P=8, rot=16, capacity=4, norm=0,
             eps=1e-6, B=1, n=4, H=2, Hk=1, D=16, dt=0)
    d.update(kw)
    return call(lib.sf_qk_norm_rope, d["x"], d["ldx"], d["q"], d["ldq"], d["s"], d["k"], d["ldk"], d["s"], d["v"],
                d["ldv"], d["s"], d["table"], d["P"], d["rot"], None, None, d["capacity"], None, None,
                c_int(d["norm"]), F32(d["eps"]), c_int(0), d["B"], d["n"], d["H"], d["Hk"], d["D"], c_int(d["dt"]),
                None)


def norm_rope_backward(lib, **kw):
    d = dict(g=A, x=A, out=A, dw=A, work=A, table=A, P=8, rot=16, norm=0, eps=1e-6, B=1, n=4, H=2, Hk=1, D=16, dt=0)
    d.update(kw)
    return call(lib.sf_qk_norm_rope_backward, d["g"], d["x"], d["table"], d["P"], d["rot"], None, None,
                c_int(d["norm"]), F32(d["eps"]), c_int(0), d["out"], d["dw"], None, d["B"], d["n"], d["H"], d["Hk"],
                d["D"], c_int(d["dt"]), d["work"], None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dt=3), INVALID, b"dtype"), (dict(norm=2), INVALID, b"norm"), (dict(B=-1), INVALID, b"batch"),
    (dict(n=-1), INVALID, b"rows"), (dict(H=0), INVALID, b"heads"), (dict(Hk=0), INVALID, b"heads"),
    (dict(D=0, rot=0), INVALID, b"D"), (dict(D=257), UNSUPPORTED, b"256"), (dict(H=4097), UNSUPPORTED, b"4096"),
    (dict(Hk=4097), UNSUPPORTED, b"4096"), (dict(B=2 ** 16, n=2 ** 15), UNSUPPORTED, b"2^30"),
    (dict(B=2 ** 62, n=2 ** 62), UNSUPPORTED, b"2^30"), (dict(rot=3), INVALID, b"even"),
    (dict(rot=18), INVALID, b"even"), (dict(rot=-2), INVALID, b"even"), (dict(table=None), INVALID, b"table"),
    (dict(P=0), INVALID, b"table"), (dict(eps=-1.0), INVALID, b"eps"), (dict(eps=float("nan")), INVALID, b"eps"),
    (dict(eps=float("inf")), INVALID, b"eps"), (dict(x=None), INVALID, b"null"),
])
def test_norm_rope_refusals(lib, kw, code, text):
    for f in (norm_rope, norm_rope_backward):
        assert f(lib, **kw) == code
        assert text in lib.sf_last_error()


@pytest.mark.parametrize("kw,text", [
    (dict(q=None), b"null"), (dict(k=None), b"null"), (dict(ldx=63), b"shorter"), (dict(ldq=31), b"shorter"),
    (dict(ldk=15), b"shorter"), (dict(ldv=15), b"shorter"), (dict(s=-1), b"stride"), (dict(capacity=-1), b"capacity"),
    (dict(v=None, ldx=47), b"shorter"),
])
def test_norm_rope_forward_refusals(lib, kw, text):
    assert norm_rope(lib, **kw) == INVALID
    assert text in lib.sf_last_error()


def test_norm_rope_backward_refusals_and_work(lib):
    for kw in (dict(g=None), dict(out=None), dict(work=None)):
        assert norm_rope_backward(lib, **kw) == INVALID
        assert b"null" in lib.sf_last_error()
    f = lib.sf_qk_norm_rope_backward_work
    assert call(f, 1, 4, 2, 1, 16, 16) > 0
    for bad in ((0, 4, 2, 1, 16, 16), (1, 0, 2, 1, 16, 16), (1, 4, 0, 1, 16, 16), (1, 4, 2, 1, 257, 0),
                (1, 4, 2, 1, 16, 17), (2 ** 62, 2 ** 62, 2, 1, 16, 16), (1, 4, 4097, 1, 16, 16)):
        assert call(f, *bad) == 0


def test_norm_rope_empty(lib):
    for kw in (dict(B=0), dict(n=0)):
        assert norm_rope(lib, x=None, q=None, k=None, **kw) == 0
        assert norm_rope_backward(lib, g=None, x=None, out=None, dw=None, work=None, **kw) == 0


def window_calls(lib, only=None, **kw):
    """The three entries, or one of them, with the same sizes and operands."""
    d = dict(Q=A, K=A, V=A, O=A, ldq=64, ldk=32, s=256, h=16, lse=A, lengths=A, B=1, H=4, Hk=2, n=4, S=8, D=16,
             window=2, sinks=1, scale=0.25, dt=2, work=A, dO=A, dQ=A, dK=A, dV=A)
    d.update(kw)
    q = lambda p: (d[p], d["ldq"], d["s"], d["h"])
    k = lambda p: (d[p], d["ldk"], d["s"], d["h"])
    tail = (d["D"], d["window"], d["sinks"], F32(d["scale"]), c_int(d["dt"]))
    heads = (d["B"], d["H"], d["Hk"], d["n"])
    if only in (None, "forward"):
        yield "forward", call(lib.sf_window_attention, *q("Q"), *k("K"), *k("V"), *q("O"), d["lse"], d["lengths"], *heads,
                              *tail, None)
    if only in (None, "backward"):
        yield "backward", call(lib.sf_window_attention_backward, *q("dO"), *q("Q"), *k("K"), *k("V"), *q("O"), d["lse"],
                               d["lengths"], *q("dQ"), *k("dK"), *k("dV"), *heads, *tail, d["work"], None)
    if only in (None, "cached"):
        yield "cached", call(lib.sf_window_attention_cached, *q("Q"), *k("K"), *k("V"), *q("O"), d["lengths"], *heads,
                             d["S"], *tail, d["work"], None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(B=-1), INVALID, b"batch"), (dict(n=-1), INVALID, b"rows"), (dict(H=0), INVALID, b"heads"),
    (dict(H=3), INVALID, b"multiple"), (dict(Hk=0), INVALID, b"kv_heads"), (dict(window=-1), INVALID, b"window"),
    (dict(sinks=-1), INVALID, b"sinks"), (dict(D=12), UNSUPPORTED, b"head size"),
    (dict(D=136), UNSUPPORTED, b"head size"), (dict(D=0), UNSUPPORTED, b"head size"),
    (dict(n=2 ** 29 + 1), UNSUPPORTED, b"2^29"), (dict(H=2 ** 21), UNSUPPORTED, b"2^24"),
    (dict(B=2 ** 25), UNSUPPORTED, b"2^24"), (dict(B=2 ** 10, H=2 ** 12, n=2 ** 10), UNSUPPORTED, b"2^24"),
    (dict(dt=3), INVALID, b"dtype"), (dict(dt=0), UNSUPPORTED, b"16-bit"),
    (dict(scale=float("nan")), INVALID, b"scale"), (dict(scale=float("inf")), INVALID, b"scale"),
    (dict(Q=None), INVALID, b"null"), (dict(K=None), INVALID, b"null"), (dict(V=None), INVALID, b"null"),
    (dict(O=None), INVALID, b"null"), (dict(ldk=8), INVALID, b"row stride"), (dict(ldq=8), INVALID, b"row stride"),
    (dict(s=-8), INVALID, b"negative stride"), (dict(h=-8), INVALID, b"negative stride"),
    (dict(Q=P(4104)), UNSUPPORTED, b"aligned"), (dict(V=P(4098)), UNSUPPORTED, b"aligned"),
    (dict(ldq=68), UNSUPPORTED, b"aligned"), (dict(s=260), UNSUPPORTED, b"aligned"),
    (dict(h=20), UNSUPPORTED, b"aligned"), (dict(ldk=2 ** 23), UNSUPPORTED, b"2^23"),
])
def test_window_refusals(lib, kw, code, text):
    for name, rc in window_calls(lib, **kw):
        assert rc == code, (name, rc, lib.sf_last_error())
        assert text in lib.sf_last_error(), (name, lib.sf_last_error())


@pytest.mark.parametrize("entry,kw,code", [
    ("backward", dict(dO=None), INVALID), ("backward", dict(dQ=None), INVALID), ("backward", dict(dK=None), INVALID),
    ("backward", dict(dV=None), INVALID), ("backward", dict(lse=None), INVALID), ("backward", dict(work=None), INVALID),
    ("backward", dict(dV=P(4104)), UNSUPPORTED), ("cached", dict(lengths=None), INVALID),
    ("cached", dict(S=0), INVALID), ("cached", dict(S=-1), INVALID), ("cached", dict(S=2 ** 29 + 1), UNSUPPORTED),
    ("cached", dict(work=None, n=1, S=2 ** 20, window=0), INVALID),
])
def test_window_refusals_of_one_entry(lib, entry, kw, code):
    assert dict(window_calls(lib, only=entry, **kw)) == {entry: code}
    assert lib.sf_last_error() != b""


def test_window_empty_and_work(lib):
    none = dict(Q=None, K=None, V=None, O=None, lse=None, lengths=None, work=None, dO=None, dQ=None, dK=None, dV=None)
    for kw in (dict(B=0), dict(n=0)):
        assert [rc for _, rc in window_calls(lib, **dict(none, **kw))] == [0, 0, 0]
    back, cached = lib.sf_window_attention_backward_work, lib.sf_window_attention_cached_work
    assert call(back, 1, 4, 2, 4, 16, 2, 1) > 0
    assert call(cached, 1, 4, 2, 1, 131072, 16, 0, 0) > 0
    for bad in ((0, 4, 2, 4), (1, 3, 2, 4), (1, 4, 2, -1), (1, 4, 2, 0), (2 ** 25, 4, 2, 4)):
        assert call(back, *bad, 16, 2, 1) == 0
        assert call(cached, *bad, 8, 16, 2, 1) == 0
    assert call(back, 1, 4, 2, 4, 12, 2, 1) == 0 and call(cached, 1, 4, 2, 1, 0, 16, 2, 1) == 0
    # any window and any number of sinks is a size
    for w in (1, 2 ** 30, 2 ** 62):
        assert call(back, 1, 4, 2, 300, 16, w, w) > 0
        assert call(cached, 1, 4, 2, 1, 131072, 16, w, w) >= 0


def gated(lib, **kw):
    d = dict(x=A, W=A, y=A, pre=A, M=4, F=16, K=16, dt=2, act=4)
    d.update(kw)
    return call(lib.sf_gated_linear, d["x"], d["W"], None, d["y"], d["pre"], d["M"], d["F"], d["K"], c_int(d["dt"]),
                c_int(d["act"]), None)


def gated_back(lib, **kw):
    d = dict(x=A, y=A, pre=A, db=A, work=A, M=4, F=16, dt=2, act=4)
    d.update(kw)
    return call(lib.sf_gated_backward, d["x"], d["pre"], d["y"], d["db"], d["M"], d["F"], c_int(d["dt"]),
                c_int(d["act"]), d["work"], None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dt=3), INVALID, b"dtype"), (dict(M=-1), INVALID, b"negative"), (dict(F=-1), INVALID, b"negative"),
    (dict(act=1), INVALID, b"activation"), (dict(act=99), INVALID, b"activation"),
    (dict(M=2 ** 30 + 1), UNSUPPORTED, b"2^30"), (dict(F=2 ** 29 + 1), UNSUPPORTED, b"2^29"),
    (dict(x=None), INVALID, b"null"), (dict(y=None), INVALID, b"null"), (dict(pre=None, dt=0), INVALID, b"null"),
])
def test_gated_refusals(lib, kw, code, text):
    for f in (gated, gated_back):
        assert f(lib, **kw) == code
        assert text in lib.sf_last_error()


def test_gated_refusals_of_one_entry(lib):
    assert gated(lib, K=-1) == INVALID and b"negative" in lib.sf_last_error()
    assert gated(lib, K=2 ** 30 + 1) == UNSUPPORTED and b"2^30" in lib.sf_last_error()
    assert gated(lib, W=None) == INVALID and b"null" in lib.sf_last_error()
    assert gated(lib, M=2 ** 20, F=2 ** 24, K=64) == UNSUPPORTED and b"2^22" in lib.sf_last_error()
    assert gated_back(lib, pre=None) == INVALID and b"null" in lib.sf_last_error()
    assert gated_back(lib, work=None) == INVALID and b"null" in lib.sf_last_error()
    work = lib.sf_gated_backward_work
    assert call(work, 4, 16) > 0 and call(work, 0, 16) == 0 and call(work, 4, 0) == 0 and call(work, -1, 16) == 0
    assert call(work, 2 ** 30 + 1, 16) == 0 and call(work, 4, 2 ** 29 + 1) == 0


def test_gated_empty(lib):
    for kw in (dict(M=0), dict(F=0)):
        assert gated(lib, x=None, W=None, y=None, pre=None, **kw) == 0
        assert gated_back(lib, x=None, y=None, pre=None, db=None, work=None, **kw) == 0


# ---- refusals of the seam -------------------------------------------------------

def fake(shape, dtype="bfloat16", dev=0):
    """A tensor without memory: the seam's checks read only its description."""
    from scaffolding_amd import _cuda_ops as g
    return g.GpuTensor(g.CudaBuffer(), tuple(shape), g.resolve_dtype(dtype), dev)


def raises(exc, f, *a, **kw):
    with pytest.raises(exc):
        f(*a, **kw)


def test_norm_rope_seam_refusals():
    from scaffolding_amd import _cuda_ops as g
    x, t, w = fake((2, 3, 64)), fake((8, 16), "float32"), fake((2, 16))
    pos, k, n = fake((2, 3), "int32"), fake((2, 5, 16)), fake((2,), "int32")
    for f, pre, post in ((g.dev_qk_norm_rope, (x,), ()), (g.dev_qk_norm_rope_backward, (x, x), ()),
                         (g.dev_qk_norm_rope_cached, (x,), (k, k, n))):
        raises(ValueError, f, *pre, 3, 1, t, *post)              # 64 columns are not 5 heads
        raises(ValueError, f, *pre, 0, 1, t, *post)
        raises(ValueError, f, *pre, 2, 1, fake((8, 15), "float32"), *post)
        raises(ValueError, f, *pre, 2, 1, fake((8, 18), "float32"), *post)
        raises(ValueError, f, *pre, 2, 1, fake((8,), "float32"), *post)
        raises(TypeError, f, *pre, 2, 1, fake((8, 16)), *post)
        raises(ValueError, f, *pre, 2, 1, fake((8, 16), "float32", 1), *post)
        raises(ValueError, f, *pre, 2, 1, t, *post, gt_weight=fake((16,)))
        raises(TypeError, f, *pre, 2, 1, t, *post, gt_weight=fake((2, 16), "float16"))
        raises(ValueError, f, *pre, 2, 1, t, *post, gt_weight=w, norm="batch")
        raises(ValueError, f, *pre, 2, 1, t, *post, gt_positions=fake((3, 2), "int32"))
        raises(TypeError, f, *pre, 2, 1, t, *post, gt_positions=fake((2, 3)))
    raises(ValueError, g.dev_qk_norm_rope, x, 2, 1, t, w, fake((2, 8)))
    raises(TypeError, g.dev_qk_norm_rope, fake((2, 3, 64), "int32"), 2, 1, t)
    raises(ValueError, g.dev_qk_norm_rope_backward, fake((2, 2, 64)), x, 2, 1, t)
    raises(TypeError, g.dev_qk_norm_rope_backward, fake((2, 3, 64), "float16"), x, 2, 1, t)
    raises(ValueError, g.dev_qk_norm_rope_cached, x, 2, 1, t, fake((2, 5, 17)), k, n)
    raises(ValueError, g.dev_qk_norm_rope_cached, x, 2, 1, t, k, fake((2, 6, 16)), n)
    raises(ValueError, g.dev_qk_norm_rope_cached, x, 2, 1, t, k, k, fake((3,), "int32"))
    raises(TypeError, g.dev_qk_norm_rope_cached, x, 2, 1, t, k, k, fake((2,)))
    raises(TypeError, g.dev_qk_norm_rope_cached, x, 2, 1, t, fake((2, 5, 16), "float16"), k, n)


def test_window_seam_refusals():
    from scaffolding_amd import _cuda_ops as g
    x, o, lse = fake((2, 3, 64)), fake((2, 3, 32)), fake((2, 2, 3), "float32")
    k, n = fake((2, 5, 16)), fake((2,), "int32")
    for f, pre, post in ((g.dev_window_attention, (x,), ()), (g.dev_window_attention_backward, (o, x, o, lse), ()),
                         (g.dev_window_attention_cached, (o, k, k, n), ())):
        raises(ValueError, f, *pre, 2, 1, 0)                     # a window of no keys
        raises(ValueError, f, *pre, 2, 1, None, -1)
        raises(ValueError, f, *pre, 0, 1)
        raises(ValueError, f, *pre, 3, 1)
    raises(ValueError, g.dev_window_attention, fake((2, 3, 112)), 3, 2)  # 3 heads do not share 2
    raises(TypeError, g.dev_window_attention, fake((2, 3, 64), "float32"), 2, 1)
    raises(ValueError, g.dev_window_attention, fake((2, 3, 48)), 2, 1)   # heads of 12
    raises(ValueError, g.dev_window_attention, fake((2, 3, 4 * 136)), 2, 1)
    raises(ValueError, g.dev_window_attention, x, 2, 1, 4, 0, None, fake((3,), "int32"))
    raises(TypeError, g.dev_window_attention, x, 2, 1, 4, 0, None, fake((2,)))
    back = g.dev_window_attention_backward
    raises(ValueError, back, fake((2, 3, 31)), x, o, lse, 2, 1)
    raises(ValueError, back, o, x, fake((2, 2, 32)), lse, 2, 1)
    raises(ValueError, back, o, x, o, fake((2, 3, 2), "float32"), 2, 1)
    raises(TypeError, back, o, x, o, fake((2, 2, 3)), 2, 1)
    raises(TypeError, back, fake((2, 3, 32), "float16"), x, o, lse, 2, 1)
    cached = g.dev_window_attention_cached
    raises(ValueError, cached, fake((3, 32)), k, k, n, 2, 1)
    raises(ValueError, cached, o, fake((2, 5, 32)), k, n, 2, 1)
    raises(TypeError, cached, o, k, fake((2, 5, 16), "float16"), n, 2, 1)
    raises(ValueError, cached, o, k, fake((2, 5, 16), dev=1), n, 2, 1)
    raises(ValueError, cached, o, k, k, fake((1,), "int32"), 2, 1)


def test_gated_seam_refusals():
    from scaffolding_amd import _cuda_ops as g
    x, w = fake((4, 16)), fake((12, 16))
    raises(ValueError, g.dev_gated_linear, x, fake((11, 16)))
    raises(ValueError, g.dev_gated_linear, x, fake((12, 15)))
    raises(ValueError, g.dev_gated_linear, x, fake((12,)))
    raises(TypeError, g.dev_gated_linear, x, fake((12, 16), "float16"))
    raises(ValueError, g.dev_gated_linear, x, w, fake((6,)))
    raises(TypeError, g.dev_gated_linear, x, w, fake((12,), "float32"))
    raises(ValueError, g.dev_gated_linear, x, w, None, "relu")
    raises(ValueError, g.dev_gated_linear, x, fake((12, 16), dev=1))
    raises(TypeError, g.dev_gated_linear, fake((4, 16), "int32"), w)
    gr, pre = fake((4, 6)), fake((4, 12))
    raises(ValueError, g.dev_gated_linear_backward, fake((4, 5)), x, w, pre)
    raises(ValueError, g.dev_gated_linear_backward, gr, x, w, fake((4, 6)))
    raises(ValueError, g.dev_gated_linear_backward, gr, fake((3, 16)), w, pre)
    raises(TypeError, g.dev_gated_linear_backward, gr, x, w, fake((4, 12), "float32"))
    raises(ValueError, g.dev_gated_linear_backward, gr, x, w, pre, True, "relu")


def test_cpu_tensors_are_refused():
    import scaffolding_amd as sf
    from scaffolding_amd.nn import functional as F
    t = sf.Tensor(np.zeros((2, 4, 64), np.float32))
    raises(RuntimeError, F.qk_norm_rope, t, 2, 1, None)
    raises(RuntimeError, F.qk_norm_rope_cached, t, 2, 1, None, t, t, t)
    raises(RuntimeError, F.qk_norm_rope_backward, t, t, 2, 1, None)
    raises(RuntimeError, F.window_attention, t, 2, 1)
    raises(RuntimeError, F.window_attention_backward, t, t, t, t, 2, 1)
    raises(RuntimeError, F.window_attention_cached, t, t, t, t, 2, 1)
    raises(RuntimeError, F.gated_linear, t, t)
    raises(RuntimeError, F.gated_linear_backward, t, t, t, t)


@pytest.mark.parametrize("length,columns", [(0, 4), (4, 0), (4, 3), (-1, 4)])
def test_rope_table_refusals(length, columns):
    from scaffolding_amd.nn import functional as F
    raises(ValueError, F.rope_table, length, columns)


def test_rope_table_on_the_host():
    """fp32 roundings of 64-bit values: half a step, 2^-24 of sizes up to 1."""
    from scaffolding_amd.nn import functional as F
    t = F.rope_table(300, 10, 500.0, device="cpu")
    assert t.shape == (300, 10)
    assert np.abs(t.numpy() - ox.rope_table(300, 10, 500.0)).max() <= 2.0 ** -24


@pytest.mark.parametrize("entry", ["backward", "cached"])
def test_window_refuses_misaligned_work(lib, entry):
    assert dict(window_calls(lib, only=entry, work=P(4104))) == {entry: INVALID}
    assert b"work" in lib.sf_last_error()


# ---- what the entries launch ------------------------------------------------------

def plan_of(lib, name, *args):
    buf = ctypes.create_string_buffer(128)
    assert call(getattr(lib, name), *args, buf, c_int(128)) == 0, lib.sf_last_error()
    return buf.value.decode()


def norm_rope_plan(lib, *sizes, values=1, backward=0):
    return plan_of(lib, "sf_qk_norm_rope_plan", *sizes, c_int(values), c_int(backward))


def test_norm_rope_plans(lib):
    sizes = 1, 17776, 30, 30, 64
    assert norm_rope_plan(lib, *sizes, 64).startswith("chunks of 8,")
    assert norm_rope_plan(lib, *sizes, 64, backward=1).startswith("chunks of 4,")
    assert norm_rope_plan(lib, *sizes, 24).startswith("chunks of 4,")
    assert norm_rope_plan(lib, *sizes, 20).startswith("chunks of 1,")
    assert norm_rope_plan(lib, 0, 4, 2, 1, 16, 16) == norm_rope_plan(lib, 4, 0, 2, 1, 16, 16) == "noop"
    buf = ctypes.create_string_buffer(8)
    plan = lambda *a: call(lib.sf_qk_norm_rope_plan, *a)
    assert plan(1, 4, 2, 1, 16, 16, c_int(1), c_int(0), None, c_int(8)) == INVALID
    assert plan(1, 4, 2, 1, 16, 16, c_int(1), c_int(0), buf, c_int(0)) == INVALID
    assert plan(1, 4, 0, 1, 16, 16, c_int(1), c_int(0), buf, c_int(8)) == INVALID
    assert plan(1, 4, 4097, 1, 16, 16, c_int(1), c_int(0), buf, c_int(8)) == UNSUPPORTED
    assert plan(1, 4, 2, 1, 257, 16, c_int(1), c_int(0), buf, c_int(8)) == UNSUPPORTED


@pytest.mark.parametrize("D,rot", [(256, 256), (256, 8), (255, 254), (129, 0), (8, 2), (1, 0)])
def test_norm_rope_of_every_size_fits_a_launch(lib, D, rot):
    """Fewer than 2^32 threads: what a launch holds."""
    for rows in (1, 1000, 2 ** 12 - 1, 2 ** 12, 2 ** 16, 2 ** 20 + 1, 2 ** 30):
        for H, Hk in ((1, 1), (1366, 1366), (4096, 1), (4096, 4096)):
            for values in (0, 1):
                for backward in (0, 1):
                    n = int(norm_rope_plan(lib, 1, rows, H, Hk, D, rot, values=values, backward=backward).split()[3])
                    assert 0 < n * 256 < 2 ** 32, (rows, H, Hk, values, backward)


def test_norm_rope_into_rows_of_its_own_input(lib):
    """With lengths a row's key goes to another row: into x that would be written
    ahead of another wave's reading, and is refused, down to one shared
    element."""
    def run(k, v, n=A, rows=4, capacity=4):
        return call(lib.sf_qk_norm_rope, P(1 << 20), 64, P(1 << 22), 32, 128, P(k), 64, 256, P(v) if v else None, 64, 256, A,
                    8, 16, None, n, capacity, None, None, c_int(0), F32(1e-6), c_int(0), 1, rows, 2, 1, 16, c_int(2), None)

    x, far = 1 << 20, 1 << 24
    size = (3 * 64 + 64) * 2  # of x
    key = (3 * 64 + 16) * 2   # of a cache
    for k, v in ((x + 64, far), (far, x + 96), (x, None), (x + size - 2, far), (x - key + 2, far), (far, x - key + 2)):
        assert run(k, v) == INVALID
        assert b"overlap" in lib.sf_last_error()
    far_rows = call(lib.sf_qk_norm_rope, P(x), 64, P(1 << 22), 32, 128, P(x + size), 2 ** 62, 2 ** 62, P(far), 64, 256, A,
                    8, 16, None, A, 2 ** 30, None, None, c_int(0), F32(1e-6), c_int(0), 2 ** 20, 4, 2, 1, 16, c_int(2), None)
    assert far_rows == INVALID and b"overlap" in lib.sf_last_error()  # 2^22 rows of x reach k


def test_gated_plans(lib):
    """Every kernel of the table has a size in the GPU's tests that chooses it."""
    import gated_cases as gc
    import test_gated_gpu as small
    for dtype, M, K, F, want in gc.LARGE:
        assert gc.plan(dtype, M, K, F) == want, (M, K, F)
    assert [gc.plan(*c) for c in small.CASES] == gc.SMALL
    assert gc.plan("bfloat16", 300, 64, 64, x=4098) == "gated 64x64 staged"
    assert gc.plan("float32", 3, 64, 64, W=4100) == "gated fp32 product, then gate"
    assert gc.plan("float16", 0, 64, 64) == gc.plan("float32", 3, 64, 0) == "noop"
    buf = ctypes.create_string_buffer(8)
    f = lib.sf_gated_linear_plan
    assert call(f, A, A, 4, 16, 16, c_int(2), None, c_int(8)) == INVALID
    assert call(f, A, A, 4, 16, 16, c_int(2), buf, c_int(0)) == INVALID
    assert call(f, A, A, 4, 16, 16, c_int(3), buf, c_int(8)) == INVALID
    assert call(f, A, A, -4, 16, 16, c_int(2), buf, c_int(8)) == INVALID
    assert call(f, A, A, 2 ** 20, 2 ** 24, 64, c_int(2), buf, c_int(8)) == UNSUPPORTED
    assert call(f, A, A, 4, 16, 16, c_int(2), buf, c_int(8)) == 0 and buf.value == b"gated 1"  # cut to the buffer


def test_window_plans(lib):
    """The sizes of the GPU's tests choose the kernels that they are there for:
    each width with 128 rows a workgroup, split and merged."""
    import window_cases as wc
    for _, B, N, H, Hk, D, window, sinks, _l, want in wc.LARGE:
        assert wc.plan(B, H, Hk, N, 0, D, window, sinks) == want
    for _, B, n, H, Hk, D, S, window, sinks, want in wc.CACHED:
        assert wc.plan(B, H, Hk, n, S, D, window, sinks) == want
    for cases, kinds in ((wc.LARGE, ["window 128 rows"]), (wc.CACHED, ["window 128 rows", "window split 1"])):
        for kind in kinds:
            assert {c[-1] for c in cases if c[-1].startswith(kind + ",")} == {
                "%s, heads up to %d" % (kind, w) for w in (64, 96, 128)}
    assert {c[-1].split()[-1] for c in wc.CACHED if "split" in c[-1] and "split 1," not in c[-1]} == {"64", "96", "128"}
    assert wc.plan(3, 6, 2, 777, 0, 72, 100, 3) == "window 64 rows, heads up to 96"
    assert wc.plan(0, 6, 2, 777, 0, 72, 100, 3) == wc.plan(3, 6, 2, 0, 9, 72, 100, 3) == "noop"
    buf, f = ctypes.create_string_buffer(8), lib.sf_window_attention_plan
    assert call(f, 1, 4, 2, 4, 8, 16, 2, 1, None, c_int(8)) == INVALID
    assert call(f, 1, 4, 2, 4, 8, 16, 2, 1, buf, c_int(0)) == INVALID
    assert call(f, 1, 3, 2, 4, 8, 16, 2, 1, buf, c_int(8)) == INVALID
    assert call(f, 1, 4, 2, 4, 8, 12, 2, 1, buf, c_int(8)) == UNSUPPORTED
    assert call(f, 1, 4, 2, 4, -1, 16, 2, 1, buf, c_int(8)) == INVALID


@pytest.mark.parametrize("first,window,sinks", [(0, None, 0), (5, 3, 2), (20, 2, 0), (0, 1, 4)])
def test_rows_in_64_bits_are_the_oracle_s(first, window, sinks):
    import window_cases as wc
    rng = np.random.default_rng(first)
    q, k, v = rng.standard_normal((6, 4)), rng.standard_normal((11, 4)), rng.standard_normal((11, 4))
    out, lse, p = ox.window_rows(q, k, v, first, window, sinks, 0.7)
    o, s, w, avg, size = wc.rows64(q, k, v, first, window, sinks, 0.7)
    assert np.abs(o - out).max() < 1e-13 and np.abs(w - p).max() < 1e-14 and (np.isinf(s) == np.isinf(lse)).all()
    there = np.isfinite(lse)
    assert np.abs(s[there] - lse[there]).max(initial=0) < 1e-13
    assert np.abs(avg - p @ np.abs(v)).max() < 1e-13


@pytest.mark.parametrize("dtype", [None, "float32"])
def test_attention_modules_refuse_fp32_where_they_are_made(dtype):
    from scaffolding_amd import nn
    raises(TypeError, nn.WindowAttention, 64, 4, device="cpu", dtype=dtype)
    raises(TypeError, nn.DecoderBlock, 64, 96, 4, device="cpu", dtype=dtype)
    assert nn.WindowAttention(64, 4, device="cpu", dtype="float16").qkv.weight.dtype.value == "float16"


@pytest.mark.parametrize("heads,kv_heads", [(2, 2 ** 31 - 1), (3, 2 ** 31 - 1), (2 ** 31 - 1, 2 ** 30), (2 ** 30, 2 ** 30)])
def test_heads_whose_sum_passes_32_bits(heads, kv_heads):
    from scaffolding_amd import _cuda_ops as g
    for f in (g.dev_qk_norm_rope, g.dev_window_attention):
        with pytest.raises(ValueError, match="projection must be"):
            f(fake((2, 3, 64)), heads, kv_heads)

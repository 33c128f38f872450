"""The 4-bit linear layer on the GPU against fp64."""
from __future__ import annotations

import ctypes
import json
import os
import subprocess
import sys

import numpy as np
import pytest

from helpers import check_bound, cu, down, gemm_bound, out_half_ulp_rel, rnd, up
from oracle import experts as ox

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
I64, P = ctypes.c_int64, ctypes.c_void_p


def raw(a, dtype):
    return cu().gputensor_from_numpy(np.ascontiguousarray(a, dtype))


def weight(rng, lead, N, K, G, dtype, zeros):
    q = rng.integers(0, 256, lead + (N, K // 2), dtype=np.uint8)
    s = np.abs(rnd(rng, lead + (K // G, N), 0.01, dtype))
    z = rng.integers(0, 16, s.shape, dtype=np.uint8) if zeros else None
    return q, s, z


def device(q, s, z, dtype):
    return raw(q, np.uint8), up(s, dtype), None if z is None else raw(z, np.uint8)


def bound(x, w, y, s, dtype, act=None):
    """The products' terms are |x| (16 + q) s with q <= 15, the group sum's
    multiples of |x| (16 + z) s: 31 |x| s each, summed in fp32 (2 K terms)."""
    K = w.shape[-1]
    top = np.swapaxes(np.asarray(s, np.float64), -1, -2)
    mag = 31.0 * np.abs(np.asarray(x, np.float64)) @ np.repeat(top, K // top.shape[-1], -1).T
    return gemm_bound(y, mag, 2 * K, dtype, act)


CASES = [
    # rows, N, K, group, zeros, activation
    (1, 1, 32, 32, False, None), (1, 4096, 4096, 128, False, "silu"), (1, 1000, 1088, 64, True, None),
    (13, 257, 1120, 32, True, "gelu"), (16, 640, 256, 256, False, None), (17, 33, 384, 128, True, "silu"),
    (32, 96, 64, 64, False, None), (33, 100, 320, 64, False, "gelu"), (64, 48, 96, 32, False, None),
    (65, 130, 512, 128, True, None), (200, 72, 2048, 1024, True, None), (100, 8300, 384, 128, False, None), (70, 4200, 8256, 64, True, None), (5, 30, 11008, 128, False, None),
    (383, 40, 128, 128, True, "silu"), (3, 64, 128, 64, True, None),
]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("M,N,K,G,zeros,act", CASES)
def test_dense(dtype, M, N, K, G, zeros, act):
    g = cu()
    rng = np.random.default_rng(M + N + K)
    x, b = rnd(rng, (M, K), 1.0, dtype), rnd(rng, (N,), 1.0, dtype)
    q, s, z = weight(rng, (), N, K, G, dtype, zeros)
    w = ox.q4_weight(q, s, z)
    xt, bt, args = up(x, dtype), up(b, dtype), device(q, s, z, dtype)
    y = x.astype(np.float64) @ w.T
    check_bound(down(g.dev_linear_q4(xt, *args)), y, bound(x, w, y, s, dtype))
    y = ox.act(y + b, act)
    check_bound(down(g.dev_linear_q4(xt, *args, bt, act)), y, bound(x, w, y, s, dtype, act))
    wt = down(g.dev_q4_expand(*args))
    check_bound(wt, w, out_half_ulp_rel(dtype) * np.abs(w) + 2.0 ** -25)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("R,E,N,K,G,zeros,act", [
    (16, 8, 300, 512, 128, False, "silu"), (1, 3, 65, 64, 32, True, None), (100, 5, 96, 320, 64, True, "gelu"),
    (400, 3, 70, 256, 128, False, None), (40, 70, 33, 128, 64, False, None), (900, 4, 50, 96, 32, True, "silu"),
])
def test_grouped(dtype, R, E, N, K, G, zeros, act):
    g = cu()
    rng = np.random.default_rng(R + E)
    off = np.concatenate([[0], np.sort(rng.integers(0, R + 1, E))])  # rows behind the last group
    x, b = rnd(rng, (R, K), 1.0, dtype), rnd(rng, (E, N), 1.0, dtype)
    q, s, z = weight(rng, (E,), N, K, G, dtype, zeros)
    w = ox.q4_weight(q, s, z)
    got = down(g.dev_linear_q4(up(x, dtype), *device(q, s, z, dtype), up(b, dtype), act, raw(off, np.int32)))
    assert (got[off[-1]:] == 0).all()
    for e in range(E):
        xe = x[off[e]:off[e + 1]]
        y = ox.act(xe.astype(np.float64) @ w[e].T + b[e], act)
        check_bound(got[off[e]:off[e + 1]], y, bound(xe, w[e], y, s[e], dtype, act), "expert %d" % e)


@pytest.mark.parametrize("E", [0, 3])
def test_many_rows_run_the_16_bit_product(E):
    """384 rows per weight and more: the weight rounded once to 16 bits."""
    g = cu()
    rng = np.random.default_rng(1)
    R, N, K = 384 * max(1, E) + 7, 96, 256
    lead = (E,) if E else ()
    x = rnd(rng, (R, K), 1.0, "bfloat16")
    q, s, z = weight(rng, lead, N, K, 64, "bfloat16", True)
    args = device(q, s, z, "bfloat16")
    wt = down(g.dev_q4_expand(*args)).astype(np.float64)
    off = [0, 500, 500, R] if E else None
    got = down(g.dev_linear_q4(up(x, "bfloat16"), *args, None, None, raw(off, np.int32) if E else None))
    y, mag = ox.grouped_linear(x, wt if E else wt[None], off or [0, R])
    check_bound(got, y, gemm_bound(y, mag, K, "bfloat16"))


@pytest.mark.parametrize("N,E", [(96, 0), (97, 0), (200, 3)])
@pytest.mark.parametrize("which", ["s", "z", "b", "y", "all"])
def test_operands_at_any_element(N, E, which):
    """Through the C ABI: scales, zero points, bias and result one element past
    an aligned address (x and q must be 16-byte aligned)."""
    g = cu()
    lib = ctypes.CDLL(os.path.join(ROOT, "scaffolding_amd", "libsfgemm.so"))
    rng = np.random.default_rng(N)
    M, K, G, dtype = 21, 320, 64, "bfloat16"
    lead = (E,) if E else ()
    x, b = rnd(rng, (M, K), 1.0, dtype), rnd(rng, lead + (N,), 1.0, dtype)
    q, s, z = weight(rng, lead, N, K, G, dtype, True)
    off = raw([0, 4, 4, 20], np.int32)
    t = dict(zip("qsz", device(q, s, z, dtype)), x=up(x, dtype), b=up(b, dtype), y=g.zeros((M, N), g.BFLOAT16))
    at, keep = {}, []
    for n, v in t.items():
        at[n] = v.data_ptr
        if n in "szby" and which in (n, "all"):
            size = np.dtype(v.dtype).itemsize
            room = g.empty((v.numel + 16,), v.dtype)
            at[n] = room.data_ptr + size
            assert lib.sf_memcpy_d2d(P(at[n]), P(v.data_ptr), ctypes.c_size_t(v.nbytes), None) == 0
            keep.append(room)
    assert lib.sf_linear_q4(P(at["x"]), P(at["q"]), P(at["s"]), P(at["z"]), P(off.data_ptr) if E else None, P(at["b"]),
                            P(at["y"]), I64(M), I64(max(1, E)), I64(N), I64(K), I64(G), 2, 1, None) == 0
    back = g.empty((M, N), g.BFLOAT16)
    assert lib.sf_memcpy_d2d(P(back.data_ptr), P(at["y"]), ctypes.c_size_t(back.nbytes), None) == 0
    want = g.dev_linear_q4(t["x"], t["q"], t["s"], t["z"], t["b"], None, off if E else None)
    assert np.array_equal(down(back), down(want))


def test_no_memory_left_for_a_16_bit_weight():
    """Many rows run the direct kernel where the 16-bit weight cannot be
    allocated."""
    r = subprocess.run([sys.executable, os.path.join(ROOT, "tests", "low_memory_q4_process.py")], capture_output=True,
                       text=True, timeout=100)
    assert r.returncode == 0, r.stdout + r.stderr
    out = json.loads(r.stdout.strip().splitlines()[-1])
    assert out["error"] == "" and out["held"] > 0 and out["same"] and 0 <= out["worst"] <= 1.0, out


def test_known_values():
    """Each nibble of each place by itself: x picks one column."""
    g = cu()
    K, N, G = 256, 16, 32
    q = np.random.default_rng(0).integers(0, 256, (N, K // 2), dtype=np.uint8)
    for dtype in ("bfloat16", "float16"):
        s = np.ones((K // G, N), np.float32) * np.arange(1, K // G + 1)[:, None]
        got = down(g.dev_linear_q4(up(np.eye(K, dtype=np.float32), dtype), raw(q, np.uint8), up(s, dtype)))
        assert np.array_equal(got, ox.q4_weight(q, s).T)


def test_values_that_are_not_finite_stay_in_their_row():
    g = cu()
    rng = np.random.default_rng(4)
    x = rnd(rng, (19, 256), 1.0, "bfloat16")
    q, s, z = weight(rng, (), 40, 256, 64, "bfloat16", True)
    w = ox.q4_weight(q, s, z)
    x[3, 7], x[17, 200] = np.nan, np.inf
    got = down(g.dev_linear_q4(up(x, "bfloat16"), *device(q, s, z, "bfloat16")))
    assert np.isnan(got[[3, 17]]).all()
    rest = np.delete(np.arange(19), [3, 17])
    y = x[rest].astype(np.float64) @ w.T
    check_bound(got[rest], y, bound(x[rest], w, y, s, "bfloat16"))


def test_no_rows_and_shapes():
    g = cu()
    q, s = raw(np.zeros((8, 32)), np.uint8), up(np.ones((1, 8)), "bfloat16")
    assert g.dev_linear_q4(up(np.zeros((0, 64)), "bfloat16"), q, s).shape == (0, 8)
    assert g.dev_linear_q4(up(np.zeros((2, 3, 64)), "bfloat16"), q, s).shape == (2, 3, 8)
    assert g.dev_linear_q4(up(np.zeros(64), "bfloat16"), q, s).shape == (8,)


def test_no_groups_give_zeros():
    """Through the C ABI: offsets of no group at all, so every row is set to 0."""
    g = cu()
    lib = ctypes.CDLL(os.path.join(ROOT, "scaffolding_amd", "libsfgemm.so"))
    x, y = up(np.ones((5, 64)), "bfloat16"), up(np.ones((5, 8)), "bfloat16")
    off = raw(np.zeros(1), np.int32)
    for bias, epi in ((None, 0), (y, 1)):
        assert lib.sf_linear_q4(P(x.data_ptr), None, None, None, P(off.data_ptr), None if bias is None else P(bias.data_ptr),
                                P(y.data_ptr), I64(5), I64(0), I64(8), I64(64), I64(32), 2, epi, None) == 0
        assert (down(y) == 0).all()
    assert g.dev_linear_q4(x, raw(np.zeros((0, 8, 32)), np.uint8), up(np.zeros((0, 2, 8)), "bfloat16"),
                           gt_offsets=off).shape == (5, 8)


def test_large_activations_keep_their_sums():
    """All x alike and positive: the offset of the packed integers is taken
    out of sums 5 times the result's."""
    g = cu()
    rng = np.random.default_rng(2)
    x = (1.0 + 0.25 * rng.random((4, 4096))).astype(np.float16).astype(np.float32)
    q, s, z = weight(rng, (), 64, 4096, 128, "float16", True)
    w = ox.q4_weight(q, s, z)
    y = x.astype(np.float64) @ w.T
    check_bound(down(g.dev_linear_q4(up(x, "float16"), *device(q, s, z, "float16"))), y, bound(x, w, y, s, "float16"))


def test_streams_and_a_captured_graph():
    g = cu()
    hip = ctypes.CDLL("libamdhip64.so.7")
    lib = ctypes.CDLL(os.path.join(ROOT, "scaffolding_amd", "libsfgemm.so"))
    rng = np.random.default_rng(3)
    M, N, K, G, E = 9, 200, 512, 64, 4
    x = up(rnd(rng, (M, K), 1.0, "bfloat16"), "bfloat16")
    q, s, z = device(*weight(rng, (E,), N, K, G, "bfloat16", True), "bfloat16")
    off = raw([0, 2, 2, 7, 9], np.int32)
    want = down(g.dev_linear_q4(x, q, s, z, None, "silu", off))
    out = g.empty((M, N), g.BFLOAT16)

    def run(st):
        return lib.sf_linear_q4(P(x.data_ptr), P(q.data_ptr), P(s.data_ptr), P(z.data_ptr), P(off.data_ptr), None,
                                P(out.data_ptr), I64(M), I64(E), I64(N), I64(K), I64(G), 2, 4, st)

    st, graph, ex = P(), P(), P()
    assert lib.sf_stream_create(ctypes.byref(st)) == 0
    assert hip.hipStreamBeginCapture(st, 0) == 0
    rc = run(st)
    assert hip.hipStreamEndCapture(st, ctypes.byref(graph)) == 0 and rc == 0
    assert hip.hipGraphInstantiate(ctypes.byref(ex), graph, None, None, ctypes.c_size_t(0)) == 0
    for _ in range(3):
        assert run(None) == 0
        g.device_synchronize()
        assert lib.sf_zero(P(out.data_ptr), ctypes.c_size_t(out.nbytes), st) == 0
        assert hip.hipGraphLaunch(ex, st) == 0 and lib.sf_stream_synchronize(st) == 0
        assert np.array_equal(down(out), want)
    hip.hipGraphExecDestroy(ex)
    hip.hipGraphDestroy(graph)
    lib.sf_stream_destroy(st)


# ---- modules ------------------------------------------------------------------------

@pytest.mark.parametrize("zeros", [False, True])
def test_linear_q4_module(zeros):
    import scaffolding_amd as sf
    from scaffolding_amd import nn

    np.random.seed(0)
    lin = nn.Linear(256, 72, dtype="bfloat16", activation="silu")
    lq = nn.LinearQ4.from_linear(lin, 64, zeros)
    x = rnd(np.random.default_rng(0), (3, 5, 256), 1.0, "bfloat16")
    y = lq(sf.Tensor(x, dtype="bfloat16", device="cuda")).numpy()
    s = lq.scales.numpy()
    w = ox.q4_weight(lq.weight.numpy(), s, lq.zeros.numpy() if zeros else None)
    flat = x.reshape(15, 256)
    y64 = ox.act(flat.astype(np.float64) @ w.T + lin.bias.numpy(), "silu")
    check_bound(y.reshape(15, 72), y64, bound(flat, w, y64, s, "bfloat16", "silu"))
    # the 4-bit weight against the weight: half a step of a seventh or a
    # fifteenth of the group's range, one more for the zero point, and the
    # scales' own rounding (times up to 15 steps)
    step = np.repeat(s.T, 64, 1).astype(np.float64)
    assert (np.abs(w - lin.weight.numpy()) <= step * (1.01 + 15 * 2.0 ** -8)).all()
    # through a state dict into a fresh module, and as fp16
    other = nn.LinearQ4(256, 72, True, 64, zeros, dtype="bfloat16", activation="silu")
    other.load_state_dict(lq.state_dict())
    assert np.array_equal(other(sf.Tensor(x, dtype="bfloat16", device="cuda")).numpy(), y)
    other.load_state_dict({n: p.numpy() for n, p in lq.state_dict().items()})
    assert np.array_equal(other(sf.Tensor(x, dtype="bfloat16", device="cuda")).numpy(), y)
    other.to(dtype="float16")
    assert other.weight.dtype is sf.uint8 and other.scales.dtype is sf.float16


def moe64(m, x, dtype):
    """MoE.forward in fp64 with the router's logits and choice as computed."""
    def w(layer):
        if layer.scales is None:
            return layer.weight.numpy()
        return ox.q4_weight(layer.weight.numpy(), layer.scales.numpy(),
                            None if layer.zeros is None else layer.zeros.numpy())
    lg = m.router(x).numpy()
    wt, e, off, slots = ox.route(lg, m.k, m.renormalize)
    rows = np.zeros((slots.size, m.dim))
    rows[slots.reshape(-1)] = np.repeat(x.numpy(), m.k, 0)
    h = ox.act(ox.grouped_linear(rows, w(m.up), off, m.up.bias.numpy())[0], "silu")
    y = ox.grouped_linear(h, w(m.down), off, m.down.bias.numpy())[0]
    return (wt[:, :, None] * y[slots]).sum(1)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("T,E,k", [(1, 4, 2), (37, 8, 2), (300, 5, 3)])
def test_moe_module(dtype, T, E, k):
    """The layer as a model calls it, in its training weights and, in 16 bits,
    in 4-bit ones: three roundings to `dtype` (hidden, expert, result) of half
    a step each and fp32 sums between, normwise."""
    import scaffolding_amd as sf
    from scaffolding_amd import nn

    np.random.seed(1)
    m = nn.MoE(64, 96, E, k, dtype=dtype)
    x = sf.Tensor(rnd(np.random.default_rng(T), (T, 64), 1.0, dtype), dtype=dtype, device="cuda")
    for quantized in (False, True):
        if quantized:
            if dtype == "float32":
                with pytest.raises(TypeError):
                    m.quantize(32)
                continue
            m.quantize(32, zeros=T == 37)
        want = moe64(m, x, dtype)
        got = m(x).numpy().astype(np.float64)
        # sums of 96 and 64 terms, with terms up to 31 / 7 of the weights'
        tol = 3 * out_half_ulp_rel(dtype) + 2 * 2 * 96 * 5 * 2.0 ** -24
        assert np.linalg.norm(got - want) <= tol * np.linalg.norm(want)


def test_moe_module_shapes_and_refusals():
    import scaffolding_amd as sf
    from scaffolding_amd import nn

    m = nn.MoE(64, 96, 4, 2, dtype="bfloat16")
    with pytest.raises(ValueError):
        m.quantize(64)  # 96 is no multiple of it: neither layer is changed
    assert m.up.scales is None and m.down.scales is None
    x = rnd(np.random.default_rng(0), (2, 3, 64), 1.0, "bfloat16")
    for quantized in (False, True):
        if quantized:
            m.quantize(32)
            with pytest.raises(RuntimeError):
                m.quantize(32)
        y = m(sf.Tensor(x, dtype="bfloat16", device="cuda")).numpy()
        flat = m(sf.Tensor(x.reshape(6, 64), dtype="bfloat16", device="cuda")).numpy()
        assert y.shape == x.shape and np.array_equal(y.reshape(6, 64), flat)
        assert m(sf.empty(0, 64, dtype="bfloat16", device="cuda")).shape == (0, 64)

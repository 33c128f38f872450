"""The causal block's operators together, as nn.DecoderBlock, a decoding loop
and a training step run them; captured and replayed; on streams; on strided,
shared and very long operands."""
from __future__ import annotations

import ctypes
import os

import numpy as np
import pytest

from helpers import check_bound, cu, down, gemm_bound, out_half_ulp_rel, quantize, rnd, up
from oracle import block as ob
from test_gated_gpu import bounds as gated_bounds
from test_normrope_gpu import steps
from test_window_gpu import backward_bound, cached_bound, check, forward_bound, ints

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
I64, P, F32 = ctypes.c_int64, ctypes.c_void_p, ctypes.c_float


@pytest.fixture(scope="module")
def lib():
    so = ctypes.CDLL(os.path.join(ROOT, "scaffolding_amd", "libsfgemm.so"))
    so.sf_last_error.restype = ctypes.c_char_p
    for name in ("sf_qk_norm_rope_backward_work", "sf_window_attention_backward_work",
                 "sf_window_attention_cached_work", "sf_gated_backward_work"):
        getattr(so, name).restype = I64
    return so


def call(f, *args):
    return f(*[I64(a) if type(a) is int else a for a in args])


def at(t, columns=0):
    """The address of a tensor's element `columns`."""
    return P(t.data_ptr + columns * (t.nbytes // max(t.numel, 1)))


# ---- the block ------------------------------------------------------------------

DIM, HID, H, HK, D, WINDOW, SINKS, ROT = 96, 160, 4, 2, 32, 12, 2, 16


def make_block(dtype, norm, seed=0):
    from scaffolding_amd import nn
    rng = np.random.default_rng(seed)
    block = nn.DecoderBlock(DIM, HID, H, HK, head_dim=D, window=WINDOW, sinks=SINKS, rotary=ROT, norm=norm,
                            max_positions=64, activation="gelu" if norm == "layer" else "silu", dtype=dtype)
    state = {}
    for name, p in block.state_dict().items():
        if "norm" in name:
            v = 0.2 * rng.standard_normal(p.shape) + (0.0 if name.endswith("bias") else 1.0)
        else:
            v = rng.standard_normal(p.shape) * p.shape[-1] ** -0.5
        state[name] = quantize(v.astype(np.float32), dtype)
    block.load_state_dict(state)
    return block, state


def rms(x, w, dtype):
    """(want, bound) of nn.RMSNorm: as a head's norm over all columns."""
    hat, r = ob.norm(x, "rms", 1e-6)
    y = hat * w
    return y, steps(x.shape[-1]) * np.abs(y) + out_half_ulp_rel(dtype) * np.abs(y) + 1e-7


def lin(x, w, dtype, res=0.0):
    x, w = np.asarray(x, np.float64), np.asarray(w, np.float64)
    lead = x.shape[:-1]
    x = x.reshape(-1, x.shape[-1])
    y, a = x @ w.T + np.reshape(res, (-1, len(w)) if np.ndim(res) else ()), np.abs(x) @ np.abs(w).T + np.abs(
        np.reshape(res, (-1, len(w)) if np.ndim(res) else ()))
    return y.reshape(*lead, -1), gemm_bound(y, a, x.shape[1], dtype).reshape(*lead, -1)


def near(got, want_bound, what):
    check_bound(got, want_bound[0], want_bound[1], what)


@pytest.mark.parametrize("dtype,norm", [("bfloat16", "rms"), ("float16", "layer")])
def test_block_over_whole_sequences(dtype, norm):
    """Every stage against the oracle on the device's own input to it, and the
    module's answer is the stages'."""
    import scaffolding_amd as sf
    from scaffolding_amd.nn import functional as F
    block, st = make_block(dtype, norm)
    rng = np.random.default_rng(1)
    B, N, lengths = 3, 40, [40, 0, 23]
    x0 = rnd(rng, (B, N, DIM), 1.0, dtype)
    x, n = sf.Tensor(x0, dtype=dtype, device="cuda"), sf.Tensor(np.array(lengths), dtype="int32", device="cuda")
    att, mlp = block.attention, block.mlp
    n1 = block.norm1(x)
    near(n1.numpy(), rms(x0, st["norm1.weight"], dtype), "norm1")
    qkv = att.qkv(n1)
    near(qkv.numpy(), lin(n1.numpy(), st["attention.qkv.weight"], dtype), "qkv")
    w, b = st["attention.norm_weight"], st.get("attention.norm_bias")
    pos = np.tile(np.arange(N), (B, 1))
    turned = F.qk_norm_rope(qkv, H, HK, att.table, att.norm_weight, att.norm_bias, norm)
    want, mag = ob.qk_norm_rope(qkv.numpy(), H, HK, att.table.numpy().astype(np.float64), pos, w, b, norm)
    check_bound(turned.numpy(), want, steps(D) * mag + out_half_ulp_rel(dtype) * np.abs(want) + 1e-7, "norm and rope")
    t = turned.numpy()
    y = F.window_attention(turned, H, HK, WINDOW, SINKS, None, n)
    want, _ = ob.window_attention(t, H, HK, WINDOW, SINKS, D ** -0.5, lengths)
    check(y.numpy(), want, forward_bound(t, H, HK, WINDOW, SINKS, D ** -0.5, dtype, lengths)[0], dtype, "attention")
    h = att.out(y, residual=x)
    near(h.numpy(), lin(y.numpy(), st["attention.out.weight"], dtype, x0), "out")
    n2 = block.norm2(h)
    near(n2.numpy(), rms(h.numpy(), st["norm2.weight"], dtype), "norm2")
    u = F.gated_linear(n2, mlp.up.weight, None, mlp.activation)
    want, pre, mag = ob.gated(n2.numpy().reshape(-1, DIM), st["mlp.up.weight"], None, mlp.activation)
    check_bound(u.numpy().reshape(-1, HID), want, gated_bounds(pre, mag, DIM, dtype, mlp.activation)[0], "gated")
    out = mlp.down(u, residual=h)
    near(out.numpy(), lin(u.numpy(), st["mlp.down.weight"], dtype, h.numpy()), "down")
    assert np.array_equal(block(x, n).numpy(), out.numpy())


@pytest.mark.parametrize("dtype,norm", [("bfloat16", "rms"), ("float16", "layer")])
def test_block_decodes_behind_its_caches(dtype, norm):
    """Prompts of unequal lengths into the caches, then tokens one at a time and
    a few at once: the caches take what the whole sequences' pass computes from
    the same rows, the attention is the oracle's over them, and the module's
    answer is the stages'."""
    import scaffolding_amd as sf
    from scaffolding_amd.nn import functional as F
    block, st = make_block(dtype, norm)
    att = block.attention
    rng = np.random.default_rng(2)
    B, cap = 3, 50
    k, v = block.cache(B, cap)
    assert k.shape == (B, cap, HK * D) and (k.numpy() == 0).all()
    seen_k, seen_v = np.zeros((B, cap, HK * D), np.float32), np.zeros((B, cap, HK * D), np.float32)
    # the first step's prompts are padded: the next ones write over the padding
    length = np.zeros(B, np.int64)
    for n, taken in [(20, [20, 7, 1]), (1, [1, 1, 1]), (1, [1, 1, 1]), (5, [5, 5, 5]), (1, [1, 1, 1])]:
        x0 = rnd(rng, (B, n, DIM), 1.0, dtype)
        x, g = sf.Tensor(x0, dtype=dtype, device="cuda"), sf.Tensor(length, dtype="int32", device="cuda")
        qkv = att.qkv(block.norm1(x))
        pos = sf.Tensor(length[:, None] + np.arange(n), dtype="int32", device="cuda")
        turned = F.qk_norm_rope(qkv, H, HK, att.table, att.norm_weight, att.norm_bias, norm, 1e-6, pos).numpy()
        q, wk, wv = np.split(turned, [H * D, (H + HK) * D], axis=2)
        for b in range(B):
            seen_k[b, length[b]:length[b] + n], seen_v[b, length[b]:length[b] + n] = wk[b], wv[b]
        got = block(x, g, (k, v))
        assert np.array_equal(k.numpy(), seen_k) and np.array_equal(v.numpy(), seen_v)
        y = F.window_attention_cached(sf.Tensor(q, dtype=dtype, device="cuda"), k, v, g, H, HK, WINDOW, SINKS)
        want = ob.window_attention_cached(q, seen_k, seen_v, length, H, HK, WINDOW, SINKS, D ** -0.5)
        check(y.numpy(), want, cached_bound(q, seen_k, seen_v, length, H, HK, WINDOW, SINKS, D ** -0.5, dtype), dtype)
        h = att.out(y, residual=x)
        assert np.array_equal(got.numpy(), block.mlp(block.norm2(h), residual=h).numpy())
        length = length + np.array(taken)


@pytest.mark.parametrize("dtype,norm,lengths", [("bfloat16", "rms", None), ("float16", "layer", [30, 0, 17])])
def test_a_training_step(dtype, norm, lengths):
    """Forward and backward through both layers of a block, each gradient
    against the formula on the device's own operands."""
    import scaffolding_amd as sf
    from scaffolding_amd.nn import functional as F
    block, st = make_block(dtype, norm)
    att, mlp = block.attention, block.mlp
    rng = np.random.default_rng(3)
    B, N, s = 3, 30, D ** -0.5
    hu = out_half_ulp_rel(dtype)
    x = sf.Tensor(rnd(rng, (B, N, DIM), 1.0, dtype), dtype=dtype, device="cuda")
    n = None if lengths is None else sf.Tensor(np.array(lengths), dtype="int32", device="cuda")
    pos = np.tile(np.arange(N), (B, 1))
    qkv = att.qkv(x)
    turned = F.qk_norm_rope(qkv, H, HK, att.table, att.norm_weight, att.norm_bias, norm)
    y, lse = F.window_attention(turned, H, HK, WINDOW, SINKS, None, n, True)
    h = att.out(y)
    u, pre = F.gated_linear(h, mlp.up.weight, None, mlp.activation, True)
    g = sf.Tensor(rnd(rng, (B, N, HID), 0.5, dtype), dtype=dtype, device="cuda")
    dh, dw, db = F.gated_linear_backward(g, h, mlp.up.weight, pre, False, mlp.activation)
    flat = [t.numpy().reshape(B * N, -1).astype(np.float64) for t in (g, h, pre)]
    wx, ww, _, d = ob.gated_backward(flat[0], flat[1], st["mlp.up.weight"], flat[2], mlp.activation)
    size = np.concatenate([np.abs(flat[0] * flat[2][:, HID:]) * 1.2, np.abs(flat[0]) * (np.abs(flat[2][:, :HID]) + 1e-3)], 1)
    sub = 2.0 ** -25 if dtype == "float16" else 0.0
    ed = 8e-6 * size + hu * np.abs(d) + sub  # d's own error, then the products' sums and one rounding
    W = np.abs(st["mlp.up.weight"]).astype(np.float64)
    for got, want, e, a in ((dh, wx, ed @ W, (np.abs(d) + ed) @ W * 2 * HID),
                            (dw, ww, ed.T @ np.abs(flat[1]), (np.abs(d) + ed).T @ np.abs(flat[1]) * B * N)):
        tol = e + 2.0 ** -23 * a
        check_bound(got.numpy().reshape(want.shape), want, tol + hu * (np.abs(want) + tol) + sub + 1e-9)
    assert db is None
    dy = sf.Tensor._wrap_gpu(cu().dev_linear_backward(dh._gpu, y._gpu, att.out.weight._gpu, False)[0])
    dt = F.window_attention_backward(dy, turned, y, lse, H, HK, WINDOW, SINKS, None, n)
    want, tol = backward_bound(dy.numpy(), turned.numpy(), H, HK, WINDOW, SINKS, s, dtype, lengths)
    check_bound(dt.numpy(), want, tol, "attention")
    dx, gw, gb = F.qk_norm_rope_backward(dt, qkv, H, HK, att.table, att.norm_weight, norm)
    (wx, ww, wb), (mx, mw, mb) = ob.qk_norm_rope_backward(dt.numpy(), qkv.numpy(), H, HK, att.table.numpy().astype(
        np.float64), pos, st["attention.norm_weight"], norm)
    terms = (steps(D) + B * N * H * 2.0 ** -24)
    check_bound(dx.numpy(), wx, 3 * steps(D) * mx + hu * np.abs(wx) + sub + 1e-7, "norm and rope")
    check_bound(gw.numpy(), ww, terms * mw + hu * np.abs(ww) + sub + 1e-7, "norm weight")
    assert (gb is None) == (norm == "rms")
    if gb is not None:
        check_bound(gb.numpy(), wb, terms * mb + hu * np.abs(wb) + sub + 1e-7, "norm bias")


def test_modules_refuse_what_they_cannot_do():
    from scaffolding_amd import nn
    ok = dict(dim=64, heads=4)
    for bad in (dict(heads=0), dict(kv_heads=3), dict(dim=65), dict(head_dim=12), dict(head_dim=136), dict(window=0),
                dict(sinks=-1), dict(rotary=3), dict(rotary=18), dict(norm="batch")):
        with pytest.raises(ValueError):
            nn.WindowAttention(**dict(ok, **bad))
    with pytest.raises(TypeError):
        nn.WindowAttention(dtype="float32", **ok)
    block = nn.DecoderBlock(64, 96, 4)
    with pytest.raises(TypeError):
        block.to(dtype="float32")
    assert all(p.dtype.value == "bfloat16" for p in block.parameters())  # nothing was moved
    block.to(dtype="float16")
    assert block.norm1.weight.dtype.value == "float16" and block.attention.table.dtype.value == "float32"
    import scaffolding_amd as sf
    x = sf.Tensor(np.zeros((1, 2, 64), np.float32), dtype="float16", device="cuda")
    with pytest.raises(ValueError):
        block(x, None, block.cache(1, 4))


# ---- captured, replayed, on streams ------------------------------------------------

class Calls:
    """Each entry on operands of its own: (call on a stream, output tensors)."""

    def __init__(self, lib, seed):
        g = cu()
        rng = np.random.default_rng(seed)
        self.kept = []

        def t(shape, dtype="bfloat16", std=1.0):
            self.kept.append(up(rnd(rng, shape, std, dtype), dtype))
            return self.kept[-1]

        def e(shape, dtype=None):
            self.kept.append(g.zeros(tuple(shape), g.BFLOAT16 if dtype is None else dtype))
            return self.kept[-1]

        def work(n):
            self.kept.append(g.empty((max(int(n) // 4, 1),)))
            return P(self.kept[-1].data_ptr)

        B, N, H, Hk, D, S = 2, 300, 4, 2, 64, 3000
        C, hd = (H + 2 * Hk) * D, H * D
        x, table, w = t((B, N, C)), t((N, D), "float32"), t((2, D))
        o1 = e((B, N, C))
        q1, k1, v1 = (P(o1.data_ptr), C, N * C), (at(o1, hd), C, N * C), (at(o1, hd + Hk * D), C, N * C)
        rope = (P(table.data_ptr), N, D, None)
        kind = (ctypes.c_int(0), F32(1e-6), ctypes.c_int(0))
        size = (B, N, H, Hk, D, ctypes.c_int(2))
        self.list = [(lambda st: call(lib.sf_qk_norm_rope, P(x.data_ptr), C, *q1, *k1, *v1, *rope, None, N,
                                      P(w.data_ptr), None, *kind, *size, st), [o1])]
        dg, dx, dw = t((B, N, C)), e((B, N, C)), e((2, D))
        w1 = work(call(lib.sf_qk_norm_rope_backward_work, B, N, H, Hk, D, D))
        self.list.append((lambda st: call(lib.sf_qk_norm_rope_backward, P(dg.data_ptr), P(x.data_ptr), *rope,
                                          P(w.data_ptr), *kind, P(dx.data_ptr), P(dw.data_ptr), None, *size, w1, st),
                          [dx, dw]))
        x2, o2, lse = t((B, N, C)), e((B, N, hd)), e((B, H, N), np.dtype(np.float32))
        parts = [(at(x2, c), C, N * C, D) for c in (0, hd, hd + Hk * D)]
        O = (P(o2.data_ptr), hd, N * hd, D)
        tail = (B, H, Hk, N, D, 100, 3, F32(0.125), ctypes.c_int(2))
        self.list.append((lambda st: call(lib.sf_window_attention, *parts[0], *parts[1], *parts[2], *O,
                                          P(lse.data_ptr), None, *tail, st), [o2, lse]))
        # the backward pass on an output and sums of its own, made beforehand
        d3, g3 = e((B, N, C)), t((B, N, hd))
        o3, l3 = g.dev_window_attention(x2, H, Hk, 100, 3, 0.125, None, True)
        self.kept += [o3, l3]
        w3 = work(call(lib.sf_window_attention_backward_work, B, H, Hk, N, D, 100, 3))
        grads = [(at(d3, c), C, N * C, D) for c in (0, hd, hd + Hk * D)]
        self.list.append((lambda st: call(lib.sf_window_attention_backward, P(g3.data_ptr), hd, N * hd, D, *parts[0],
                                          *parts[1], *parts[2], P(o3.data_ptr), hd, N * hd, D, P(l3.data_ptr), None,
                                          *grads[0], *grads[1], *grads[2], *tail, w3, st), [d3]))
        q4, k4, v4, o4 = t((B, 1, hd)), t((B, S, Hk * D)), t((B, S, Hk * D)), e((B, 1, hd))
        n4 = ints([S - 1, 1700])
        self.kept.append(n4)
        need = call(lib.sf_window_attention_cached_work, B, H, Hk, 1, S, D, 0, 0)
        assert need > 0  # split, with a merge
        w4 = work(need)
        self.list.append((lambda st: call(lib.sf_window_attention_cached, P(q4.data_ptr), hd, hd, D, P(k4.data_ptr),
                                          Hk * D, S * Hk * D, D, P(v4.data_ptr), Hk * D, S * Hk * D, D, P(o4.data_ptr),
                                          hd, hd, D, P(n4.data_ptr), B, H, Hk, 1, S, D, 0, 0, F32(0.125),
                                          ctypes.c_int(2), w4, st), [o4]))
        M, K, Fh = 70, 256, 200
        x5, W5, y5, p5 = t((M, K)), t((2 * Fh, K), std=0.1), e((M, Fh)), e((M, 2 * Fh))
        self.list.append((lambda st: call(lib.sf_gated_linear, P(x5.data_ptr), P(W5.data_ptr), None, P(y5.data_ptr),
                                          P(p5.data_ptr), M, Fh, K, ctypes.c_int(2), ctypes.c_int(4), st), [y5, p5]))
        g6, p6, d6, b6 = t((M, Fh)), t((M, 2 * Fh)), e((M, 2 * Fh)), e((2 * Fh,))
        w6 = work(call(lib.sf_gated_backward_work, M, Fh))
        self.list.append((lambda st: call(lib.sf_gated_backward, P(g6.data_ptr), P(p6.data_ptr), P(d6.data_ptr),
                                          P(b6.data_ptr), M, Fh, ctypes.c_int(2), ctypes.c_int(4), w6, st), [d6, b6]))
        y7 = e((4, Fh))
        self.list.append((lambda st: call(lib.sf_gated_linear, P(x5.data_ptr), P(W5.data_ptr), None, P(y7.data_ptr),
                                          None, 4, Fh, K, ctypes.c_int(2), ctypes.c_int(4), st), [y7]))

    def outputs(self):
        return [down(t) for _, out in self.list for t in out]


def test_captured_and_replayed(lib):
    """All entries in one graph: every replay gives the eager results, with
    eager calls of the same entries on other operands between the replays."""
    g = cu()
    hip = ctypes.CDLL("libamdhip64.so.7")
    a, other = Calls(lib, 0), Calls(lib, 1)
    for run, _ in a.list:
        assert run(None) == 0
    want = a.outputs()
    st, graph, ex = P(), P(), P()
    assert lib.sf_stream_create(ctypes.byref(st)) == 0
    g.device_synchronize()
    assert hip.hipStreamBeginCapture(st, 0) == 0
    rcs = [run(st) for run, _ in a.list]
    assert hip.hipStreamEndCapture(st, ctypes.byref(graph)) == 0 and rcs == [0] * len(rcs)
    assert hip.hipGraphInstantiate(ctypes.byref(ex), graph, None, None, ctypes.c_size_t(0)) == 0
    for _ in range(3):
        for run, _o in other.list:
            assert run(None) == 0
        g.device_synchronize()
        for _r, out in a.list:
            for t in out:
                assert lib.sf_zero(P(t.data_ptr), ctypes.c_size_t(t.nbytes), st) == 0
        assert hip.hipGraphLaunch(ex, st) == 0 and lib.sf_stream_synchronize(st) == 0
        for y, w in zip(a.outputs(), want):
            assert np.array_equal(y, w)
    hip.hipGraphExecDestroy(ex)
    hip.hipGraphDestroy(graph)
    lib.sf_stream_destroy(st)


def test_two_streams_at_once(lib):
    """Both streams run every entry several times, each with operands and
    workspaces of its own, and get what the default stream got."""
    g = cu()
    sets = [Calls(lib, 2), Calls(lib, 3)]
    want = []
    for s in sets:
        for run, _ in s.list:
            assert run(None) == 0
        want.append(s.outputs())
    streams = [P(), P()]
    for st in streams:
        assert lib.sf_stream_create(ctypes.byref(st)) == 0
    g.device_synchronize()
    for s, st in zip(sets, streams):
        for _r, out in s.list:
            for t in out:
                assert lib.sf_zero(P(t.data_ptr), ctypes.c_size_t(t.nbytes), st) == 0
    for _ in range(5):
        for i in range(len(sets[0].list)):
            for s, st in zip(sets, streams):
                assert s.list[i][0](st) == 0
    for st in streams:
        assert lib.sf_stream_synchronize(st) == 0
    for s, w in zip(sets, want):
        for y, e in zip(s.outputs(), w):
            assert np.array_equal(y, e)
    for st in streams:
        lib.sf_stream_destroy(st)


# ---- strided, shared and very long operands ------------------------------------------

@pytest.mark.parametrize("dtype,norm,D,R", [("bfloat16", "rms", 64, 64), ("float32", "layer", 36, 10)])
def test_norm_rope_in_place(lib, dtype, norm, D, R):
    """q, k and v the input's own columns; the gradient over its own input."""
    rng = np.random.default_rng(4)
    B, N, H, Hk = 2, 77, 3, 2
    C, hd, code = (H + 2 * Hk) * D, H * D, {"float32": 0, "bfloat16": 2}[dtype]
    x0, g0, w0 = rnd(rng, (B, N, C), 1.0, dtype), rnd(rng, (B, N, C), 1.0, dtype), rnd(rng, (2, D), 1.0, dtype)
    x, w, t = up(x0, dtype), up(w0, dtype), cu().gputensor_from_numpy(ob.rope_table(N, R).astype(np.float32))
    want = down(cu().dev_qk_norm_rope(x, H, Hk, t, w, None, norm))
    dx, dw, _ = cu().dev_qk_norm_rope_backward(up(g0, dtype), x, H, Hk, t, w, norm)
    kind = (ctypes.c_int(norm == "layer"), F32(1e-6), ctypes.c_int(0))
    size = (B, N, H, Hk, D, ctypes.c_int(code))
    rope = (P(t.data_ptr), N, R, None)
    g, gw = up(g0, dtype), cu().empty((2, D), x.dtype)
    work = cu().empty((call(lib.sf_qk_norm_rope_backward_work, B, N, H, Hk, D, R) // 4,))
    assert call(lib.sf_qk_norm_rope_backward, P(g.data_ptr), P(x.data_ptr), *rope, P(w.data_ptr), *kind,
                P(g.data_ptr), P(gw.data_ptr), None, *size, P(work.data_ptr), None) == 0
    assert np.array_equal(down(g), down(dx)) and np.array_equal(down(gw), down(dw))
    args = (*rope, None, N, P(w.data_ptr), None, *kind, *size, None)
    assert call(lib.sf_qk_norm_rope, P(x.data_ptr), C, P(x.data_ptr), C, N * C, at(x, hd), C, N * C,
                at(x, hd + Hk * D), C, N * C, *args) == 0
    assert np.array_equal(down(x), want)
    # without v the values are not read: rows of queries and keys alone
    x2 = up(x0[..., :(H + Hk) * D], dtype)
    c2 = (H + Hk) * D
    assert call(lib.sf_qk_norm_rope, P(x2.data_ptr), c2, P(x2.data_ptr), c2, N * c2, at(x2, hd), c2, N * c2, None, 0, 0,
                *args) == 0
    assert np.array_equal(down(x2), want[..., :c2])


def test_gate_gradient_over_its_own_input(lib):
    rng = np.random.default_rng(5)
    M, Fh = 33, 77
    g, pre = up(rnd(rng, (M, Fh), 1.0, "float16"), "float16"), up(rnd(rng, (M, 2 * Fh), 1.0, "float16"), "float16")
    out = cu().empty((M, 2 * Fh), np.dtype(np.float16))
    work = cu().empty((call(lib.sf_gated_backward_work, M, Fh) // 4,))
    db = [cu().empty((2 * Fh,), np.dtype(np.float16)) for _ in range(2)]
    tail = (M, Fh, ctypes.c_int(1), ctypes.c_int(4))
    for bias in (db[0], None):
        assert call(lib.sf_gated_backward, P(g.data_ptr), P(pre.data_ptr), P(out.data_ptr),
                    None if bias is None else P(bias.data_ptr), *tail, P(work.data_ptr), None) == 0
        want = down(out) if bias is not None else want
        assert np.array_equal(down(out), want)  # the same with the sums and without
    assert call(lib.sf_gated_backward, P(g.data_ptr), P(pre.data_ptr), P(pre.data_ptr), P(db[1].data_ptr), *tail,
                P(work.data_ptr), None) == 0
    assert np.array_equal(down(pre), want) and np.array_equal(down(db[0]), down(db[1]))


@pytest.mark.parametrize("dtype,M,F", [("bfloat16", 1, 1), ("float32", 17, 9), ("float16", 700, 37), ("bfloat16", 3, 2500),
                                       ("bfloat16", 300, 2056), ("float32", 9000, 8), ("bfloat16", 1500, 4097)])
def test_sums_of_the_gate_gradient(lib, dtype, M, F):
    """The bias's gradient: fp32 sums (2^-24 a term, over M terms) of terms that
    carry a few fp32 steps of sizes up to 1.2 |g up| and |g act|, one
    rounding."""
    rng = np.random.default_rng(M)
    code, hu = {"float32": 0, "float16": 1, "bfloat16": 2}[dtype], out_half_ulp_rel(dtype)
    g0, p0 = rnd(rng, (M, F), 1.0, dtype), rnd(rng, (M, 2 * F), 1.0, dtype)
    g, pre = up(g0, dtype), up(p0, dtype)
    out, db = cu().empty((M, 2 * F), g.dtype), cu().empty((2 * F,), g.dtype)
    work = cu().empty((call(lib.sf_gated_backward_work, M, F) // 4,))
    assert call(lib.sf_gated_backward, P(g.data_ptr), P(pre.data_ptr), P(out.data_ptr), P(db.data_ptr), M, F,
                ctypes.c_int(code), ctypes.c_int(4), P(work.data_ptr), None) == 0
    _, _, want, d = ob.gated_backward(g0, np.zeros((M, 1)), np.zeros((2 * F, 1)), p0, "silu")
    size = np.concatenate([np.abs(g0 * p0[:, F:]) * 1.2, np.abs(g0) * (np.abs(p0[:, :F]) + 1e-3)], 1).astype(np.float64)
    sub = 2.0 ** -25 if dtype == "float16" else 1e-30
    check_bound(down(out), d, 8e-6 * size + hu * np.abs(d) + sub, "gradient")
    tol = ((8e-6 + M * 2.0 ** -24) * size).sum(0)
    check_bound(down(db), want, tol + hu * (np.abs(want) + tol) + sub, "sums")


def place(B, N, heads, D, order, gap):
    """(strides of row, batch, head; elements) of a (B, N, heads, D) operand,
    rows of one head together or heads of one row together, with gaps."""
    ld, head = (D + gap, (N + 1) * (D + gap)) if order == "heads" else (heads * D + gap, D)
    batch = heads * head + gap if order == "heads" else N * ld + gap
    return (ld, batch, head), B * batch + gap


def put(a, strides, total, dtype):
    """a (B, N, heads, D) laid out with the strides, NaN between."""
    ld, batch, head = strides
    flat = np.full(total, np.nan, np.float32)
    B, N, heads, D = a.shape
    for b in range(B):
        for h in range(heads):
            for i in range(N):
                o = b * batch + h * head + i * ld
                flat[o:o + D] = a[b, i, h]
    return up(flat, dtype)


def take(t, strides, shape):
    ld, batch, head = strides
    flat, out = down(t), np.empty(shape, np.float32)
    mask = np.ones(len(flat), bool)
    B, N, heads, D = shape
    for b in range(B):
        for h in range(heads):
            for i in range(N):
                o = b * batch + h * head + i * ld
                out[b, i, h] = flat[o:o + D]
                mask[o:o + D] = False
    return out, flat[mask]


@pytest.mark.parametrize("D,window", [(64, 20), (72, 0)])
def test_window_operands_laid_out_anyhow(lib, D, window):
    """Each operand with strides of its own and NaN in the gaps: the packed
    call's results bit for bit, and nothing written between the rows."""
    rng = np.random.default_rng(6)
    dtype, B, N, H, Hk, sinks, scale = "bfloat16", 2, 150, 4, 2, 3, 0.11
    x = rnd(rng, (B, N, (H + 2 * Hk) * D), 1.0, dtype)
    g = rnd(rng, (B, N, H * D), 1.0, dtype)
    gx = up(x, dtype)
    o, lse = cu().dev_window_attention(gx, H, Hk, window or None, sinks, scale, None, True)
    want_dx = down(cu().dev_window_attention_backward(up(g, dtype), gx, o, lse, H, Hk, window or None, sinks, scale))
    heads = x.reshape(B, N, H + 2 * Hk, D)
    cut = {"Q": heads[:, :, :H], "K": heads[:, :, H:H + Hk], "V": heads[:, :, H + Hk:],
           "dO": g.reshape(B, N, H, D)}
    lay, t = {}, {}
    for i, (name, a) in enumerate(cut.items()):
        lay[name], total = place(B, N, a.shape[2], D, ("heads", "rows")[i % 2], 8 * (i + 1))
        t[name] = put(a, lay[name], total, dtype)
    for i, (name, n) in enumerate((("O", H), ("dQ", H), ("dK", Hk), ("dV", Hk))):
        lay[name], total = place(B, N, n, D, ("heads", "rows")[i % 2], 8 * (4 - i))
        t[name] = up(np.full(total, np.nan, np.float32), dtype)
    arg = lambda name: (P(t[name].data_ptr), *lay[name])
    size = (B, H, Hk, N, D, window, sinks, F32(scale), ctypes.c_int(2))
    l2 = cu().empty((B, H, N))
    assert call(lib.sf_window_attention, *arg("Q"), *arg("K"), *arg("V"), *arg("O"), P(l2.data_ptr), None, *size,
                None) == 0
    work = cu().empty((call(lib.sf_window_attention_backward_work, B, H, Hk, N, D, window, sinks) // 4,))
    assert call(lib.sf_window_attention_backward, *arg("dO"), *arg("Q"), *arg("K"), *arg("V"), *arg("O"),
                P(l2.data_ptr), None, *arg("dQ"), *arg("dK"), *arg("dV"), *size, P(work.data_ptr), None) == 0
    assert np.array_equal(down(l2), down(lse))
    dx = want_dx.reshape(B, N, H + 2 * Hk, D)
    for name, want in (("O", down(o).reshape(B, N, H, D)), ("dQ", dx[:, :, :H]), ("dK", dx[:, :, H:H + Hk]),
                       ("dV", dx[:, :, H + Hk:])):
        got, gaps = take(t[name], lay[name], want.shape)
        assert np.array_equal(got, want), name
        assert np.isnan(gaps).all(), name


def test_one_cache_for_several_sequences(lib):
    """Sequences that share a prompt: batch strides of 0."""
    rng = np.random.default_rng(7)
    B, H, Hk, D, S = 3, 4, 2, 64, 200
    q, k, v = (rnd(rng, s, 1.0, "float16") for s in ((B, 1, H * D), (1, S, Hk * D), (1, S, Hk * D)))
    n = ints([S - 1, 100, 5])
    want = down(cu().dev_window_attention_cached(up(q, "float16"), up(np.repeat(k, B, 0), "float16"),
                                                 up(np.repeat(v, B, 0), "float16"), n, H, Hk, 50, 2, 0.125))
    gq, gk, gv, out = up(q, "float16"), up(k, "float16"), up(v, "float16"), cu().empty((B, 1, H * D), np.dtype(np.float16))
    need = call(lib.sf_window_attention_cached_work, B, H, Hk, 1, S, D, 50, 2)
    work = cu().empty((max(need // 4, 1),))
    assert call(lib.sf_window_attention_cached, P(gq.data_ptr), H * D, H * D, D, P(gk.data_ptr), Hk * D, 0, D,
                P(gv.data_ptr), Hk * D, 0, D, P(out.data_ptr), H * D, H * D, D, P(n.data_ptr), B, H, Hk, 1, S, D, 50, 2,
                F32(0.125), ctypes.c_int(1), P(work.data_ptr), None) == 0
    assert np.array_equal(down(out), want)


@pytest.mark.parametrize("n", [1, 150])
def test_offsets_past_32_bits(lib, n):
    """Caches of 2^31 elements and more: the new rows go to their ends, and the
    attention reads the first rows and those at the end."""
    rng = np.random.default_rng(8)
    dtype, H, Hk, D, window, sinks = "bfloat16", 8, 8, 128, 70, 3
    S = 2 ** 21 + 400
    assert S * Hk * D > 2 ** 31
    k, v = (cu().zeros((1, S, Hk * D), cu().BFLOAT16) for _ in range(2))
    length = S - n - 5
    x = rnd(rng, (1, n, 3 * H * D), 1.0, dtype)
    rows = rnd(rng, (2, window + sinks, Hk * D), 1.0, dtype)
    for cache, r in ((k, rows[0]), (v, rows[1])):
        for first, part in ((0, r[:sinks]), (length - window, r[sinks:])):
            src = up(part, dtype)
            assert lib.sf_memcpy_d2d(P(cache.data_ptr + first * Hk * D * 2), P(src.data_ptr),
                                     ctypes.c_size_t(src.nbytes), None) == 0
    g = ints([length])
    table = cu().gputensor_from_numpy(ob.rope_table(n + 4, D).astype(np.float32))
    pos = np.arange(n)[None] + 2
    q = cu().dev_qk_norm_rope_cached(up(x, dtype), H, Hk, table, k, v, g, None, None, "rms", 1e-6, ints(pos))
    y = down(cu().dev_window_attention_cached(q, k, v, g, H, Hk, window, sinks, 0.09))
    turned = down(cu().dev_qk_norm_rope(up(x, dtype), H, Hk, table, None, None, "rms", 1e-6, ints(pos)))
    wq, wk, wv = np.split(turned, 3, axis=2)
    assert np.array_equal(down(q), wq)
    # the same rows in a short cache: first ones, a window, the new ones
    sk, sv = (np.concatenate([r[None], w], 1) for r, w in ((rows[0], wk), (rows[1], wv)))
    args = (wq, sk, sv, [window + sinks], H, Hk, window, sinks, 0.09)
    check(y, ob.window_attention_cached(*args), cached_bound(*args, dtype), dtype)
    tail = np.empty((n, Hk * D), np.uint16)
    assert lib.sf_memcpy_d2h(P(tail.ctypes.data), P(k.data_ptr + length * Hk * D * 2), ctypes.c_size_t(tail.nbytes),
                             None) == 0
    assert np.array_equal((tail.astype(np.uint32) << 16).view(np.float32), wk[0])


def test_batches_more_than_32_bits_apart(lib):
    """Two sequences of one packed operand, 2^31 elements between them, and
    gradients laid out alike."""
    rng = np.random.default_rng(9)
    B, N, H, Hk, D, window, sinks = 2, 100, 2, 1, 64, 30, 2
    C, hd, apart = (H + 2 * Hk) * D, H * D, 2 ** 31 + 64
    x, g = rnd(rng, (B, N, C), 1.0, "bfloat16"), rnd(rng, (B, N, hd), 1.0, "bfloat16")
    gx, gg = up(x, "bfloat16"), up(g, "bfloat16")
    o, lse = cu().dev_window_attention(gx, H, Hk, window, sinks, 0.125, None, True)
    dx = cu().dev_window_attention_backward(gg, gx, o, lse, H, Hk, window, sinks, 0.125)

    def spread(t, columns):
        far = cu().empty((apart + N * columns,), cu().BFLOAT16)
        if t is not None:
            for b in range(B):
                assert lib.sf_memcpy_d2d(P(far.data_ptr + b * apart * 2), P(t.data_ptr + b * N * columns * 2),
                                         ctypes.c_size_t(N * columns * 2), None) == 0
        return far

    def gather(far, columns):
        t = cu().empty((B, N, columns), cu().BFLOAT16)
        for b in range(B):
            assert lib.sf_memcpy_d2d(P(t.data_ptr + b * N * columns * 2), P(far.data_ptr + b * apart * 2),
                                     ctypes.c_size_t(N * columns * 2), None) == 0
        return down(t)

    fx, fg, fo, fd = spread(gx, C), spread(gg, hd), spread(None, hd), spread(None, C)
    parts = lambda t: [(at(t, c), C, apart, D) for c in (0, hd, hd + Hk * D)]
    size = (B, H, Hk, N, D, window, sinks, F32(0.125), ctypes.c_int(2))
    l2 = cu().empty((B, H, N))
    pq, pk, pv = parts(fx)
    O = (P(fo.data_ptr), hd, apart, D)
    assert call(lib.sf_window_attention, *pq, *pk, *pv, *O, P(l2.data_ptr), None, *size, None) == 0
    work = cu().empty((call(lib.sf_window_attention_backward_work, B, H, Hk, N, D, window, sinks) // 4,))
    dq, dk, dv = parts(fd)
    assert call(lib.sf_window_attention_backward, P(fg.data_ptr), hd, apart, D, *pq, *pk, *pv, *O, P(l2.data_ptr), None,
                *dq, *dk, *dv, *size, P(work.data_ptr), None) == 0
    assert np.array_equal(gather(fo, hd), down(o)) and np.array_equal(down(l2), down(lse))
    assert np.array_equal(gather(fd, C), down(dx))


@pytest.mark.parametrize("M,K,F", [(1, 4, 1), (3, 2416, 200), (16, 260, 37), (5, 16, 16), (2, 516, 20), (16, 4, 64)])
@pytest.mark.parametrize("act,bias", [("silu", True), ("gelu", False), (None, True)])
def test_gated_fp32_of_few_rows(M, K, F, act, bias):
    rng = np.random.default_rng(M + K)
    x, W = rnd(rng, (M, K), 1.0, "float32"), rnd(rng, (2 * F, K), K ** -0.5, "float32")
    b = rnd(rng, (2 * F,), 0.5, "float32") if bias else None
    want, pre, mag = ob.gated(x, W, b, act)
    ty, tp = gated_bounds(pre, mag, K, "float32", act)
    y, p = cu().dev_gated_linear(up(x, "float32"), up(W, "float32"), up(b, "float32") if bias else None, act, True)
    check_bound(down(y), want, ty, "y")
    check_bound(down(p), pre, tp, "pre")


def test_sequences_and_caches_past_the_table_are_refused():
    import scaffolding_amd as sf
    from scaffolding_amd import nn
    att = nn.WindowAttention(64, 4, max_positions=6, dtype="float16")
    with pytest.raises(ValueError):
        att.cache(1, 7)
    with pytest.raises(ValueError):
        att(sf.Tensor(np.zeros((1, 7, 64), np.float32), dtype="float16", device="cuda"))
    assert att(sf.Tensor(np.zeros((1, 6, 64), np.float32), dtype="float16", device="cuda")).shape == (1, 6, 64)
    assert att.cache(1, 6)[0].shape == (1, 6, 64)


@pytest.mark.parametrize("M,F,K", [(2 ** 20 + 300, 8, 1032), (2 ** 20 + 300, 8, 1027), (20, 2 ** 18 + 40, 2056),
                                   (3, 2 ** 18 + 40, 2056), (3, 2 ** 18 + 40, 2051)])
def test_gated_operands_past_2_gib(lib, M, F, K):
    """The last rows of x, or of W's gate and up halves, lie past 2^31 bytes;
    what is before them is 0."""
    rng = np.random.default_rng(M)
    tall = M > F
    assert (M if tall else 2 * F) * K * 2 > 2 ** 31
    m, f = (50, F) if tall else (M, 30)  # rows that are not 0, the last ones
    x0, W0 = rnd(rng, (m, K), 1.0, "bfloat16"), rnd(rng, (2 * f, K), K ** -0.5, "bfloat16")
    x, W = cu().zeros((M, K), cu().BFLOAT16), cu().zeros((2 * F, K), cu().BFLOAT16)
    for dst, row, part in ((x, M - m, x0), (W, F - f, W0[:f]), (W, 2 * F - f, W0[f:])):
        src = up(part, "bfloat16")
        assert lib.sf_memcpy_d2d(P(dst.data_ptr + row * K * 2), P(src.data_ptr), ctypes.c_size_t(src.nbytes), None) == 0
    y, pre = cu().dev_gated_linear(x, W, None, "silu", True)
    want, wp, mag = ob.gated(x0, W0, None, "silu")
    ty, tp = gated_bounds(wp, mag, K, "bfloat16", "silu")
    y, pre = down(y), down(pre)
    check_bound(y[M - m:, F - f:], want, ty, "y")
    check_bound(np.concatenate([pre[M - m:, F - f:F], pre[M - m:, 2 * F - f:]], 1), wp, tp, "pre")
    assert not y[:M - m].any() and not y[:, :F - f].any()

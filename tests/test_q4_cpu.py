"""The 4-bit linear layer without a GPU: quantize_q4, and the refusals of the
C entries and the seam."""
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
    return so


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("shape,group", [((5, 64), 32), ((3, 4, 256), 128), ((1, 32), 32)])
def test_quantize(shape, group, zeros):
    from scaffolding_amd.nn import functional as F
    rng = np.random.default_rng(0)
    w = rng.standard_normal(shape).astype(np.float32)
    w[..., :group] *= 1e-3
    q, s, z = F.quantize_q4(w, group, zeros)
    assert q.dtype == np.uint8 and q.shape == shape[:-1] + (shape[-1] // 2,)
    assert s.shape == shape[:-2] + (shape[-1] // group, shape[-2]) and (z is None) == (not zeros)
    back = ox.q4_weight(q, s, z)
    step = np.repeat(np.swapaxes(s, -1, -2), group, -1)
    # half a step; a rounded zero point moves the ends by up to half a step more
    assert (np.abs(back - w) <= step * (1.001 if zeros else 0.501)).all()
    if not zeros:  # the largest of a group is kept
        top = np.abs(w.reshape(-1, group)).max(1)
        assert np.allclose(np.abs(back.reshape(-1, group)).max(1), top, rtol=1e-6)


def test_quantize_zero_groups_and_refusals():
    from scaffolding_amd.nn import functional as F
    for zeros in (False, True):
        q, s, z = F.quantize_q4(np.zeros((2, 64), np.float32), 32, zeros)
        assert (ox.q4_weight(q, s, z) == 0).all() and (s == 0).all()
    for bad in (np.zeros((2, 48)), np.zeros(64), np.full((2, 64), np.nan), np.full((2, 64), np.inf)):
        with pytest.raises(ValueError):
            F.quantize_q4(bad, 32)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dt=7), -2, b"dtype"), (dict(dt=0), -3, b"F16"), (dict(R=-1), -2, b"negative"), (dict(N=-1), -2, b"negative"),
    (dict(G=16), -3, b"group"), (dict(G=96), -3, b"group"), (dict(G=0), -3, b"group"), (dict(G=-32), -3, b"group"),
    (dict(K=100), -2, b"multiple"), (dict(E=2), -2, b"offsets"), (dict(E=1025, o=A), -3, b"groups"),
    (dict(epi=6), -2, b"epilogue"), (dict(epi=1), -2, b"bias"), (dict(x=None), -2, b"null"), (dict(q=None), -2, b"null"),
    (dict(s=None), -2, b"null"), (dict(y=None), -2, b"null"), (dict(x=P(4104)), -3, b"aligned"),
    (dict(q=P(4097)), -3, b"aligned"), (dict(R=2 ** 31), -3, b"2^31"), (dict(R=2 ** 30), -3, b"tiles"),
    (dict(K=2 ** 25), -3, b"2^25"),
])
def test_refusals(lib, kw, code, text):
    d = dict(x=A, q=A, s=A, o=None, y=A, R=4, E=1, N=16, K=128, G=64, dt=2, epi=0)
    d.update(kw)
    assert lib.sf_linear_q4(d["x"], d["q"], d["s"], None, d["o"], None, d["y"], I64(d["R"]), I64(d["E"]), I64(d["N"]),
                            I64(d["K"]), I64(d["G"]), d["dt"], d["epi"], None) == code
    assert text in lib.sf_last_error()


def test_empty_and_expand_refusals(lib):
    assert lib.sf_linear_q4(None, None, None, None, None, None, None, I64(0), I64(1), I64(8), I64(32), I64(32), 2, 0, None) == 0
    assert lib.sf_linear_q4(None, None, None, None, None, None, None, I64(4), I64(1), I64(0), I64(32), I64(32), 2, 0, None) == 0

    def expand(q=A, s=A, w=A, E=1, N=8, K=64, G=32, dt=2):
        return lib.sf_q4_expand(q, s, None, w, I64(E), I64(N), I64(K), I64(G), dt, None)

    assert expand(q=None, s=None, w=None, N=0) == 0 and expand(q=None, s=None, w=None, K=0) == 0
    assert expand(dt=0) == -3 and expand(G=48) == -3 and expand(K=48) == -2 and expand(w=None) == -2
    assert expand(w=P(4098)) == -3


def fake(shape, dtype="bfloat16", dev=0):
    from scaffolding_amd import _cuda_ops as g
    return g.GpuTensor(g.CudaBuffer(), tuple(shape), g.resolve_dtype(dtype), dev)


def test_seam_refusals():
    from scaffolding_amd import _cuda_ops as g
    x, q, s = fake((4, 128)), fake((16, 64), "uint8"), fake((2, 16))

    def no(exc, *a, **k):
        with pytest.raises(exc):
            g.dev_linear_q4(*a, **k)

    no(TypeError, fake((4, 128), "float32"), q, fake((2, 16), "float32"))
    no(TypeError, fake((4, 128), "float16"), q, s)
    no(TypeError, x, fake((16, 64)), s)
    no(ValueError, fake((4, 64)), q, s)
    no(ValueError, x, q, fake((16, 2)))
    no(ValueError, x, q, fake((8, 16)))          # groups of 16
    no(ValueError, x, q, fake((0, 16)))
    no(ValueError, x, q, fake((3, 16)))
    no(ValueError, x, q, s, fake((2, 15), "uint8"))
    no(TypeError, x, q, s, fake((2, 16)))
    no(ValueError, x, q, s, None, fake((15,)))
    no(TypeError, x, q, s, None, fake((16,), "float16"))
    no(ValueError, x, q, s, None, None, "relu")
    no(ValueError, x, q, s, None, None, None, fake((3,), "int32"))  # offsets need one weight per group
    no(ValueError, x, fake((16, 64), "uint8", 1), s)
    qe, se = fake((2, 16, 64), "uint8"), fake((2, 2, 16))
    no(ValueError, x, qe, se)
    no(ValueError, x, qe, se, None, None, None, fake((2,), "int32"))
    no(TypeError, x, qe, se, None, None, None, fake((3,)))
    no(ValueError, fake((2, 2, 128)), qe, se, None, None, None, fake((3,), "int32"))
    for bad in ((q, fake((2, 15))), (fake((64,), "uint8"), s), (q, fake((3, 16)))):
        with pytest.raises(ValueError):
            g.dev_q4_expand(*bad)
    with pytest.raises(TypeError):
        g.dev_q4_expand(q, fake((2, 16), "float32"))


def test_module_refusals():
    import scaffolding_amd as sf
    from scaffolding_amd import nn
    from scaffolding_amd.nn import functional as F
    with pytest.raises(ValueError):
        nn.LinearQ4(100, 8, group=32)
    with pytest.raises(ValueError):
        nn.LinearQ4(96, 8, group=48)
    with pytest.raises(ValueError):
        nn.MoE(8, 8, 4, 5)
    t = sf.Tensor(np.zeros((4, 128), np.float16))
    with pytest.raises(RuntimeError):
        F.linear_q4(t, t, t)


def test_a_4_bit_layer_is_16_bit():
    """Scales and activations are float16 or bfloat16: any other type is
    refused where the layer is made or moved, and nothing is changed."""
    import scaffolding_amd as sf
    from scaffolding_amd import nn
    with pytest.raises(TypeError):
        nn.LinearQ4(64, 8, group=32, device="cpu", dtype="float32")
    with pytest.raises(TypeError):
        nn.LinearQ4(64, 8, group=32, device="cpu", dtype="int32")
    lin = nn.Linear(64, 8, device="cpu")
    with pytest.raises(TypeError):
        nn.LinearQ4.from_linear(lin, 32)
    lq = nn.LinearQ4.from_linear(lin, 32, dtype="float16")
    assert lq.scales.dtype is sf.float16 and lq.bias.dtype is sf.float16 and lq.weight.dtype is sf.uint8
    seq = nn.Sequential(nn.Linear(8, 64, device="cpu"), lq)
    for m in (lq, seq):
        with pytest.raises(TypeError):
            m.to(dtype="float32")
    assert seq._modules["0"].weight.dtype is sf.float32 and lq.scales.dtype is sf.float16
    with pytest.raises(TypeError):
        seq.to(dtype="uint8")
    seq.to(device="cpu")
    seq.to(dtype="float16")
    assert seq._modules["0"].weight.dtype is sf.float16 and lq.weight.dtype is sf.uint8


def test_a_quantized_expert_layer_is_16_bit():
    import scaffolding_amd as sf
    from scaffolding_amd import nn
    m = nn.MoE(64, 32, 3, 2, device="cpu", dtype="float16")
    m.to(dtype="float32").to(dtype="float16")
    m.quantize(32)
    with pytest.raises(TypeError):
        m.to(dtype="float32")
    assert {p.dtype for p in m.parameters()} == {sf.float16, sf.uint8}
    m.to(device="cpu", dtype="float16")


def test_quantize_needs_whole_bytes():
    """Two columns share a byte: an odd number of them is refused."""
    from scaffolding_amd.nn import functional as F
    for shape, group in (((2, 3), 3), ((2, 1), 1), ((4, 5, 15), 5)):
        with pytest.raises(ValueError):
            F.quantize_q4(np.ones(shape, np.float32), group)
    q, s, z = F.quantize_q4(np.ones((2, 6), np.float32), 3)
    # 7 steps of 1 / 7, which fp32 holds to half a step of it
    assert q.shape == (2, 3) and (np.abs(ox.q4_weight(q, s) - 1) <= 2.0 ** -24).all()


@pytest.mark.parametrize("zeros", [False, True])
def test_quantize_of_the_largest_weights(zeros):
    """A group's range may pass the largest fp32 number; its step does not."""
    from scaffolding_amd.nn import functional as F
    top = np.finfo(np.float32).max
    w = np.tile(np.array([top, -top, 0.0, top / 2], np.float32), (2, 8))
    with np.errstate(all="raise", under="ignore"):
        q, s, z = F.quantize_q4(w, 32, zeros)
    assert np.isfinite(s).all()
    back = ox.q4_weight(q, s, z)
    step = np.repeat(np.swapaxes(s, -1, -2), 32, -1).astype(np.float64)
    assert (np.abs(back - w) <= step * (1.001 if zeros else 0.501)).all()


# ---- which variant runs ------------------------------------------------------------

def test_the_gpu_tests_reach_every_variant():
    """On 256 CUs: each tile and wave count, dense and grouped, with scale
    groups of 32, 64 and 128, with and without zero points, and scales that
    pass through LDS in one part and in several."""
    from q4_cases import DENSE, GROUPED, PARTS, plan, variant_cases
    seen = set()
    for R, E, N, K, G, zeros, cols, waves in variant_cases():
        assert plan(R, E, N, K, G, zeros).startswith("q4 16x%d %d waves," % (cols, waves)), (R, E, N, K, G)
        seen.add((cols, waves, E > 0, min(G, 128), zeros))
    assert set(DENSE) == set(GROUPED) == {(c, w) for c, w, *_ in seen}
    assert len(seen) == 6 * 2 * 3 * 2
    parts = set()
    for R, E, N, K, G, zeros, n in PARTS:
        p = plan(R, E, N, K, G, zeros)
        assert p.endswith("scales in %d" % n), (p, R, N, K)
        parts.add((p.split("x")[1].split()[0], min(G, 128), n > 1))
    assert {c for c, _, many in parts if many} == {"16", "32", "64"} and {g for _, g, many in parts if many} == {32, 64, 128}


def test_plan_refusals(lib):
    buf = ctypes.create_string_buffer(96)

    def plan(R=4, E=1, N=16, K=128, G=64, zeros=0, grouped=0, to=buf, n=96):
        return lib.sf_linear_q4_plan(I64(R), I64(E), I64(N), I64(K), I64(G), zeros, grouped, to, n)

    assert plan() == 0 and buf.value == b"q4 16x16 8 waves, scales in 1"
    assert plan(R=0) == 0 and buf.value == b"noop"
    assert plan(n=4) == 0 and buf.value == b"q4 "
    assert plan(to=None) == -2 and plan(n=0) == -2 and plan(E=2) == -2 and plan(G=48) == -3 and plan(K=100) == -2
    assert plan(E=0, grouped=1) == 0

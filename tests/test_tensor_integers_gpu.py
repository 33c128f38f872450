"""Integer storage types on the device: exact both ways, and refused by every
operator that computes."""
from __future__ import annotations

import numpy as np
import pytest

from helpers import cu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["int32", "uint8"])
@pytest.mark.parametrize("n", [0, 1, 3, 17, 100003])
def test_values_are_kept(dtype, n):
    import scaffolding_amd as sf
    info = np.iinfo(dtype)
    v = np.random.default_rng(n).integers(info.min, info.max, n, dtype=dtype, endpoint=True)
    t = sf.Tensor(v, dtype=dtype, device="cuda")
    assert t.dtype is sf.dtype(dtype) and t.numpy().dtype == np.dtype(dtype) and np.array_equal(t.numpy(), v)
    assert np.array_equal(t.cpu().numpy(), v) and t.cpu().dtype is sf.dtype(dtype)
    assert np.array_equal(t.cpu().to("cuda").reshape(1, -1).numpy().reshape(-1), v)
    z = sf.zeros(n, dtype=dtype)
    assert z.dtype is sf.dtype(dtype) and (z.numpy() == 0).all()
    if n:
        cu().dev_copy(t._gpu, z._gpu)
        assert np.array_equal(z.numpy(), v)


@pytest.mark.parametrize("values,dtype", [([300], "uint8"), ([1.5], "int32"), ([2 ** 31], "int32"), ([np.inf], "uint8")])
def test_values_out_of_range_are_refused(values, dtype):
    import scaffolding_amd as sf
    from scaffolding_amd import nn
    with pytest.raises(TypeError):
        sf.Tensor(values, dtype=dtype, device="cuda")
    m = nn.Module()
    m.q = nn.Parameter(np.zeros(1, dtype), False, dtype, "cuda")
    with pytest.raises(TypeError):
        m.load_state_dict({"q": np.array(values)})
    assert m.q.numpy().tolist() == [0] and m.q.dtype is sf.dtype(dtype)


@pytest.mark.parametrize("dtype", ["int32", "uint8"])
def test_operators_refuse_integers(dtype):
    import scaffolding_amd as sf
    g = cu()
    t = sf.Tensor(np.ones((4, 4)).astype(dtype), dtype=dtype, device="cuda")._gpu
    v = sf.Tensor(np.ones(4).astype(dtype), dtype=dtype, device="cuda")._gpu
    f = g.gputensor_from_numpy(np.ones((4, 4), np.float32))
    q = g.dev_reshape(t, (1, 4, 4))
    for call in (lambda: g.dev_matmul(t, t), lambda: g.dev_matmul_nt(t, t), lambda: g.dev_matmul_tn(t, t),
                 lambda: g.dev_batched_matmul(q, q), lambda: g.dev_matmul(f, t), lambda: g.dev_linear_forward(t, t, v),
                 lambda: g.dev_linear_forward(f, f, v), lambda: g.dev_linear_backward(t, t, t),
                 lambda: g.dev_sum_dim(t, 0), lambda: g.dev_softmax(t), lambda: g.dev_silu(t), lambda: g.dev_gelu(t),
                 lambda: g.dev_muls(t, 2.0), lambda: g.dev_dropout(t, 0.5), lambda: g.dev_add(t, t),
                 lambda: g.dev_bias_add(t, v), lambda: g.dev_layer_norm(t), lambda: g.dev_rms_norm(t),
                 lambda: g.dev_cast(t, np.float32), lambda: g.dev_cast(f, np.dtype(dtype)),
                 lambda: g.dev_scaled_dot_product_attention(q, q, q), lambda: g.dev_softmax_masked(f, t),
                 lambda: g.dev_route_topk(t, 1), lambda: g.dev_grouped_linear(t, q, v)):
        with pytest.raises((TypeError, ValueError)):
            call()

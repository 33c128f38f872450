"""Functional ops of the path (reference nn/functional.py).

  linear                          reference nn/functional.py:374-395
  silu / gelu (tanh)              reference nn/functional.py:37-89
  softmax                         reference nn/functional.py:113-145
  dropout                         reference nn/functional.py:231-238
  scaled_dot_product_attention    reference nn/functional.py:298-369
  route_topk, dispatch_rows,
  combine_rows, grouped_linear    experts, with their gradients (no reference
                                  counterparts)
  quantize_q4, linear_q4          4-bit weights (no reference counterpart)
  rope_table, qk_norm_rope        per-head norms and rotation, over a sequence
                                  or into a cache, with their gradient (no
                                  reference counterpart)
  window_attention                causal attention over a window and sinks, over
                                  a sequence or a cache, with its gradient (no
                                  reference counterpart)
  gated_linear                    gated feed-forward projections, with their
                                  gradient (no reference counterpart)

GPU only; results carry no grad_fn (as the reference's GPU branches).
"""
from __future__ import annotations

import math
from typing import NamedTuple

import numpy as np

from .. import _cuda_ops as _cuops
from ..tensor import Tensor, _gpu_only
from .layers import _linear, _on


def linear(input: Tensor, weight: Tensor, bias: Tensor | None = None,
           activation: str | None = None) -> Tensor:
    return _linear(input, weight, bias, activation)


def silu(input: Tensor) -> Tensor:
    if input._gpu is None:
        _gpu_only("silu")
    return Tensor._wrap_gpu(_cuops.dev_silu(input._gpu), input._device)


def gelu(input: Tensor, approximate: str = "tanh") -> Tensor:
    if input._gpu is None:
        _gpu_only("gelu")
    if approximate != "tanh":
        raise NotImplementedError("only the tanh approximation is on the device path")
    return Tensor._wrap_gpu(_cuops.dev_gelu(input._gpu), input._device)


def softmax(input: Tensor, dim: int = -1, dtype=None) -> Tensor:
    if input._gpu is None:
        _gpu_only("softmax")
    if dtype is not None:
        raise NotImplementedError("softmax(dtype=...) is not on the device path")
    return Tensor._wrap_gpu(_cuops.dev_softmax(input._gpu, dim), input._device)


def dropout(input: Tensor, p: float = 0.5, training: bool = True) -> Tensor:
    """Zeroes each element with probability p and scales the rest by
    1 / (1 - p) (reference nn/functional.py:231-238, GPU branch
    dev_dropout); identity when not training or p == 0.  Each call draws
    the next stream of the device random state (scaffolding_amd.cuda
    .manual_seed); the reference's GPU branch passes seed 0 every call."""
    if not training or p == 0.0:
        return input
    if input._gpu is None:
        _gpu_only("dropout")
    seed, offset = _cuops.next_random_stream()
    out, _ = _cuops.dev_dropout(input._gpu, p, seed, offset, False)
    return Tensor._wrap_gpu(out, input._device)


def scaled_dot_product_attention(q: Tensor, k: Tensor, v: Tensor, attn_mask=None,
                                 dropout_p: float = 0.0, scale: float | None = None) -> Tensor:
    """softmax(scale * q k^T + attn_mask) v, scale defaulting to 1/sqrt(head
    size).  16-bit inputs with a head size that is a multiple of 8 up to 128
    run as one fused launch, with or without a mask (sf_attention_masked: the
    scores never reach memory); other inputs take three launches: a
    strided-batched QK^T with the scale in its epilogue, a row softmax with
    the additive mask folded in, and a strided-batched PV.  The reference's GPU path
    (nn/functional.py:310-321) runs a Python loop of per-head SGEMMs, a
    scale pass, the softmax and a batched SGEMM, and sends a masked call to
    its host branch (:339-341: scores += mask, NumPy broadcasting); here
    the mask (a Tensor on the device, or a host array or CPU Tensor, which
    is uploaded) is applied on the device with the same broadcasting.
    dropout_p > 0 drops attention weights before PV as the reference's GPU
    branch does (:317-318), on the three-launch path, with the next stream
    of the device random state (see dropout)."""
    if q._gpu is None or k._gpu is None or v._gpu is None:
        _gpu_only("scaled_dot_product_attention")
    seed, offset = _cuops.next_random_stream() if dropout_p > 0.0 else (0, 0)
    mask = None
    if attn_mask is not None:
        if isinstance(attn_mask, Tensor):
            mask = attn_mask._gpu if attn_mask._gpu is not None else attn_mask.numpy()
        else:
            mask = attn_mask
    d = q.shape[-1]
    s = (1.0 / math.sqrt(d)) if scale is None else float(scale)
    out = _cuops.dev_scaled_dot_product_attention(q._gpu, k._gpu, v._gpu, s, mask, dropout_p, seed, offset)
    return Tensor._wrap_gpu(out, q._device)


class Routing(NamedTuple):
    """What route_topk gives: weights (fp32) and experts (int32), both (..., k),
    in descending order of the logits; offsets (int32, (E + 1,)) and slots
    (int32, (..., k)): with the choices ordered by expert, within one by token,
    slots holds each one's place, and expert e's places are offsets[e] to
    offsets[e + 1] - 1."""
    weights: Tensor
    experts: Tensor
    offsets: Tensor
    slots: Tensor
    renormalize: bool = True


def _device_of(op: str, first: Tensor, *others) -> int:
    """The device that `first` lives on, made current; every operand on a GPU."""
    for t in (first,) + others:
        if t is not None and t._gpu is None:
            _gpu_only(op)
    dev = first._gpu.device_id
    _cuops.set_device(dev)
    return dev


def route_topk(logits: Tensor, k: int, renormalize: bool = True) -> Routing:
    """Sends each token to the k experts of its largest logits (..., E):
    weights softmax(logits) of the chosen in fp32, divided by their sum with
    `renormalize`.  Equal logits go to the lower index, NaN counts above every
    number, and a token whose logits are all -inf gets weights 0.  E <= 1024,
    k <= min(E, 16)."""
    _device_of("route_topk", logits)
    out = _cuops.dev_route_topk(logits._gpu, k, renormalize)
    return Routing(*(Tensor._wrap_gpu(t, logits._device) for t in out), renormalize)


def route_topk_backward(grad_weights: Tensor, logits: Tensor, routing: Routing) -> Tensor:
    """Gradient of route_topk's logits, in their dtype, from the fp32 gradient
    of its weights (the choice itself has none)."""
    dev = _device_of("route_topk_backward", logits, grad_weights, routing.weights, routing.experts)
    out = _cuops.dev_route_topk_backward(_on(grad_weights, dev), logits._gpu, _on(routing.weights, dev),
                                         _on(routing.experts, dev), routing.renormalize)
    return Tensor._wrap_gpu(out, logits._device)


def dispatch_rows(input: Tensor, slots: Tensor) -> Tensor:
    """Tokens (..., D) in expert order: (T k, D) rows, rows[slots[t, j]] =
    input[t].  Its gradient is combine_rows without weights."""
    dev = _device_of("dispatch_rows", input, slots)
    return Tensor._wrap_gpu(_cuops.dev_dispatch_rows(input._gpu, _on(slots, dev)), input._device)


def combine_rows(rows: Tensor, slots: Tensor, weights: Tensor | None = None) -> Tensor:
    """Tokens from rows in expert order: sum over j of weights[t, j]
    rows[slots[t, j]] (fp32, one rounding); weights fp32 (..., k), None: 1."""
    dev = _device_of("combine_rows", rows, slots, weights)
    return Tensor._wrap_gpu(_cuops.dev_combine_rows(rows._gpu, _on(slots, dev), _on(weights, dev)), rows._device)


def combine_rows_backward(grad: Tensor, rows: Tensor, slots: Tensor, weights: Tensor) -> tuple[Tensor, Tensor]:
    """(grad_rows, grad_weights) of combine_rows; grad_weights is fp32."""
    dev = _device_of("combine_rows_backward", rows, grad, slots, weights)
    out = _cuops.dev_combine_rows_backward(_on(grad, dev), rows._gpu, _on(slots, dev), _on(weights, dev))
    return tuple(Tensor._wrap_gpu(t, rows._device) for t in out)


def grouped_linear(input: Tensor, weight: Tensor, offsets: Tensor, bias: Tensor | None = None,
                   activation: str | None = None) -> Tensor:
    """A linear layer with one weight per group of rows, in one launch:
    act(input[r] W[e]^T + b[e]) for the rows r of group e.  input (R, K),
    weight (E, N, K), bias (E, N); group e is the rows offsets[e] to
    offsets[e + 1] - 1 of the int32 tensor offsets (E + 1,), ascending from 0,
    and may be empty; rows from offsets[E] on give 0.  The sizes are read on
    the device: offsets may come straight from route_topk."""
    dev = _device_of("grouped_linear", input, weight, offsets, bias)
    out = _cuops.dev_grouped_linear(input._gpu, _on(weight, dev), _on(offsets, dev), _on(bias, dev), activation)
    return Tensor._wrap_gpu(out, input._device)


def grouped_linear_backward(grad: Tensor, input: Tensor, weight: Tensor, offsets: Tensor, has_bias: bool = True,
                            activation: str | None = None, pre: Tensor | None = None
                            ) -> tuple[Tensor, Tensor, Tensor | None]:
    """(grad_input, grad_weight, grad_bias or None) of grouped_linear; with an
    activation, `pre` is the layer's output without it."""
    dev = _device_of("grouped_linear_backward", input, grad, weight, offsets, pre)
    out = _cuops.dev_grouped_linear_backward(_on(grad, dev), input._gpu, _on(weight, dev), _on(offsets, dev),
                                             has_bias, activation, _on(pre, dev))
    return tuple(None if t is None else Tensor._wrap_gpu(t, input._device) for t in out)


def quantize_q4(weight, group: int = 128, zeros: bool = False):
    """A weight (..., N, K) (array or Tensor) in 4 bits, as NumPy arrays: (q
    uint8 (..., N, K / 2), scales float32 (..., K / group, N), zero points
    uint8 of the scales' shape or None), for linear_q4.  Symmetric by default
    (values -7 .. 7 times max|w| / 7 of the group, so the largest is kept);
    with `zeros` the group's range, widened to hold 0, is cut into 15 steps.
    Runs on the host, once, when a model is loaded."""
    w = weight.numpy() if isinstance(weight, Tensor) else np.asarray(weight)
    w = w.astype(np.float32)
    if w.ndim < 2 or group < 1 or w.shape[-1] % group != 0:
        raise ValueError("quantize_q4: weight %s does not divide into groups of %d" % (w.shape, group))
    if w.shape[-1] % 2:
        raise ValueError("quantize_q4: two columns share a byte, %d is odd" % w.shape[-1])
    if not np.isfinite(w).all():
        raise ValueError("quantize_q4: the weight has values that are not finite")
    g = w.reshape(w.shape[:-1] + (w.shape[-1] // group, group))
    if zeros:
        low, high = np.minimum(g.min(-1), 0.0), np.maximum(g.max(-1), 0.0)
        with np.errstate(over="ignore"):
            scale = (high - low) / 15.0
        scale = np.where(np.isfinite(scale), scale, high / 15.0 - low / 15.0)  # a range past the largest number
        zero = np.rint(-low / np.where(scale == 0.0, 1.0, scale))
    else:
        scale = np.abs(g).max(-1) / 7.0
        zero = np.full(scale.shape, 8.0, np.float32)
    q = np.rint(g / np.where(scale == 0.0, 1.0, scale)[..., None]) + zero[..., None]
    q = np.clip(q, 0, 15).astype(np.uint8).reshape(w.shape)
    packed = q[..., 0::2] | (q[..., 1::2] << 4)
    return (packed, np.ascontiguousarray(np.swapaxes(scale, -1, -2).astype(np.float32)),
            np.ascontiguousarray(np.swapaxes(zero, -1, -2).astype(np.uint8)) if zeros else None)


def linear_q4(input: Tensor, qweight: Tensor, scales: Tensor, zeros: Tensor | None = None,
              bias: Tensor | None = None, activation: str | None = None, offsets: Tensor | None = None) -> Tensor:
    """A linear layer with a 4-bit weight W[n, k] = (q[n, k] - z[k // G, n])
    s[k // G, n]: input (..., K) fp16 or bf16, qweight uint8 (N, K / 2) with
    the even column in the low four bits, scales (K / G, N) of the input's
    dtype, zeros uint8 (K / G, N) or None for 8, G = 32, 64 or a multiple of
    128 (quantize_q4 makes them).  With offsets (see grouped_linear), one
    weight, scales, zeros and bias per group of rows, a leading E each."""
    dev = _device_of("linear_q4", input, qweight, scales, zeros, bias, offsets)
    out = _cuops.dev_linear_q4(input._gpu, _on(qweight, dev), _on(scales, dev), _on(zeros, dev), _on(bias, dev),
                               activation, _on(offsets, dev))
    return Tensor._wrap_gpu(out, input._device)


def rope_table(length: int, columns: int, base: float = 10000.0, device=None) -> Tensor:
    """The rotation's table for positions 0 .. length - 1, fp32 (length,
    columns): cos(p base^(-2 j / columns)) for j < columns / 2, then the sines.
    Angles are formed in 64 bits on the host, once; any table of this layout
    will do (other spacings, several axes)."""
    if length < 1 or columns < 2 or columns % 2:
        raise ValueError("rope_table: needs a length and an even number of columns, got %d and %d" % (length, columns))
    turn = np.arange(length)[:, None] * float(base) ** (-np.arange(0, columns, 2) / columns)
    return Tensor(np.concatenate([np.cos(turn), np.sin(turn)], 1).astype(np.float32), device=device or "cuda")


def qk_norm_rope(qkv: Tensor, heads: int, kv_heads: int, table: Tensor | None, weight: Tensor | None = None,
                 bias: Tensor | None = None, norm: str = "rms", eps: float = 1e-6, positions: Tensor | None = None,
                 interleaved: bool = False) -> Tensor:
    """Norms each query and key head of a packed projection (B, N, (heads + 2
    kv_heads) D) (norm 'rms' or 'layer'; weight and bias (2, D): queries, keys)
    and rotates its first R columns by the token's row of `table` (P, R) (see
    rope_table): columns (j, j + R / 2), or (2 j, 2 j + 1) with `interleaved`.
    Token i takes row i, or positions[b, i] (int32 (B, N)); a position that the
    table does not have gives NaN.  Values go through.  D <= 256."""
    dev = _device_of("qk_norm_rope", qkv, table, weight, bias, positions)
    out = _cuops.dev_qk_norm_rope(qkv._gpu, heads, kv_heads, _on(table, dev), _on(weight, dev), _on(bias, dev), norm,
                                  eps, _on(positions, dev), interleaved)
    return Tensor._wrap_gpu(out, qkv._device)


def qk_norm_rope_cached(qkv: Tensor, heads: int, kv_heads: int, table: Tensor | None, k_cache: Tensor,
                        v_cache: Tensor, lengths: Tensor, weight: Tensor | None = None, bias: Tensor | None = None,
                        norm: str = "rms", eps: float = 1e-6, positions: Tensor | None = None,
                        interleaved: bool = False) -> Tensor:
    """qk_norm_rope of n new tokens a sequence, (B, n, ...), behind the
    lengths[b] (int32 (B,)) that the caches (B, capacity, kv_heads D) hold: row
    i stands at lengths[b] + i, its keys and values are written there (rows past
    the capacity are dropped), and the queries (B, n, heads D) are returned.
    `lengths` stays as it is."""
    dev = _device_of("qk_norm_rope_cached", qkv, table, k_cache, v_cache, lengths, weight, bias, positions)
    _written_on("qk_norm_rope_cached", dev, k_cache, v_cache)
    out = _cuops.dev_qk_norm_rope_cached(qkv._gpu, heads, kv_heads, _on(table, dev), k_cache._gpu, v_cache._gpu,
                                         _on(lengths, dev), _on(weight, dev), _on(bias, dev), norm, eps,
                                         _on(positions, dev), interleaved)
    return Tensor._wrap_gpu(out, qkv._device)


def _written_on(op: str, dev: int, *written) -> None:
    for t in written:  # a copy would take the writes
        if t._gpu.device_id != dev:
            raise ValueError("%s: the caches must be on the device of the new tokens" % op)


def qk_norm_rope_backward(grad: Tensor, qkv: Tensor, heads: int, kv_heads: int, table: Tensor | None,
                          weight: Tensor | None = None, norm: str = "rms", eps: float = 1e-6,
                          positions: Tensor | None = None, interleaved: bool = False, has_bias: bool | None = None
                          ) -> tuple[Tensor, Tensor, Tensor | None]:
    """(grad_qkv, grad_weight (2, D), grad_bias (2, D) or None) of qk_norm_rope,
    qkv being its input; the bias's with has_bias, or where that is None for
    norm 'layer'."""
    dev = _device_of("qk_norm_rope_backward", qkv, grad, table, weight, positions)
    out = _cuops.dev_qk_norm_rope_backward(_on(grad, dev), qkv._gpu, heads, kv_heads, _on(table, dev),
                                           _on(weight, dev), norm, eps, _on(positions, dev), interleaved, has_bias)
    return tuple(None if t is None else Tensor._wrap_gpu(t, qkv._device) for t in out)


def window_attention(qkv: Tensor, heads: int, kv_heads: int, window: int | None = None, sinks: int = 0,
                     scale: float | None = None, lengths: Tensor | None = None, return_lse: bool = False):
    """Causal attention of a packed projection (B, N, (heads + 2 kv_heads) D) ->
    (B, N, heads D): token i sees the tokens j <= i with j > i - window (None:
    all of them) or j < sinks; heads / kv_heads query heads share a key head;
    scale defaults to 1 / sqrt(D).  lengths (int32 (B,)) ends each sequence:
    nothing behind it is seen, and rows behind it give 0.  return_lse: (output,
    lse), the rows' log-sums fp32 (B, heads, N), for
    window_attention_backward.  float16 or bfloat16, D a multiple of 8 up to
    128; one launch, heads read in place."""
    dev = _device_of("window_attention", qkv, lengths)
    out = _cuops.dev_window_attention(qkv._gpu, heads, kv_heads, window, sinks, scale, _on(lengths, dev), return_lse)
    if return_lse:
        return tuple(Tensor._wrap_gpu(t, qkv._device) for t in out)
    return Tensor._wrap_gpu(out, qkv._device)


def window_attention_backward(grad: Tensor, qkv: Tensor, out: Tensor, lse: Tensor, heads: int, kv_heads: int,
                              window: int | None = None, sinks: int = 0, scale: float | None = None,
                              lengths: Tensor | None = None) -> Tensor:
    """grad_qkv of window_attention, in qkv's layout, from grad (B, N, heads
    D); out and lse are what it gave with return_lse for the same arguments."""
    dev = _device_of("window_attention_backward", qkv, grad, out, lse, lengths)
    dx = _cuops.dev_window_attention_backward(_on(grad, dev), qkv._gpu, _on(out, dev), _on(lse, dev), heads, kv_heads,
                                              window, sinks, scale, _on(lengths, dev))
    return Tensor._wrap_gpu(dx, qkv._device)


def window_attention_cached(q: Tensor, k_cache: Tensor, v_cache: Tensor, lengths: Tensor, heads: int, kv_heads: int,
                            window: int | None = None, sinks: int = 0, scale: float | None = None) -> Tensor:
    """window_attention of n new tokens a sequence, q (B, n, heads D), over
    caches (B, capacity, kv_heads D) to which qk_norm_rope_cached has added
    theirs: token i of sequence b stands at lengths[b] + i (int32 (B,), the
    lengths before these tokens)."""
    dev = _device_of("window_attention_cached", q, k_cache, v_cache, lengths)
    out = _cuops.dev_window_attention_cached(q._gpu, _on(k_cache, dev), _on(v_cache, dev), _on(lengths, dev), heads,
                                             kv_heads, window, sinks, scale)
    return Tensor._wrap_gpu(out, q._device)


def gated_linear(input: Tensor, weight: Tensor, bias: Tensor | None = None, activation: str | None = "silu",
                 return_pre: bool = False):
    """The up side of a gated feed-forward layer: act(input Wg^T + bg) * (input
    Wu^T + bu), weight (2 F, K) holding Wg's rows, then Wu's, bias (2 F,)
    likewise; (..., K) -> (..., F).  One launch; two for some 16-bit layers of
    many rows and for fp32 past 16 rows.  return_pre: (output, pre), pre (..., 2
    F) the two projections, for gated_linear_backward."""
    dev = _device_of("gated_linear", input, weight, bias)
    out = _cuops.dev_gated_linear(input._gpu, _on(weight, dev), _on(bias, dev), activation, return_pre)
    if return_pre:
        return tuple(Tensor._wrap_gpu(t, input._device) for t in out)
    return Tensor._wrap_gpu(out, input._device)


def gated_linear_backward(grad: Tensor, input: Tensor, weight: Tensor, pre: Tensor, has_bias: bool = False,
                          activation: str | None = "silu") -> tuple[Tensor, Tensor, Tensor | None]:
    """(grad_input, grad_weight, grad_bias or None) of gated_linear; `pre` from
    return_pre (or linear of the same operands)."""
    dev = _device_of("gated_linear_backward", input, grad, weight, pre)
    out = _cuops.dev_gated_linear_backward(_on(grad, dev), input._gpu, _on(weight, dev), _on(pre, dev), has_bias,
                                           activation)
    return tuple(None if t is None else Tensor._wrap_gpu(t, input._device) for t in out)

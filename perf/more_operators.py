"""Performance cases of the operators of a causal transformer block.

  norm_rope  per-head norm of queries and keys with the position rotation in
             the same pass, over a packed projection or into a cache, and its
             backward pass
  window     causal attention over a sliding window of keys and a few first
             ones (sinks), queries sharing key heads: over whole sequences, its
             backward pass, and over a cache for a few new tokens
  gated      a gated feed-forward layer's two projections, activation and
             product, and its backward pass

``own`` says which side runs: the plain form in elementary torch operations
(fp32, one rounding at the end), or the package's entry points on the package's
own tensors, which ``prepare`` fills with the same values in the same layout.

  listed()                the named cases
  draw(rng)               one more case of the ranges the listed ones stand for
  prepare(case, seed)     inputs on the GPU, from the seed
  run(state)              one pass and its outputs
  work(case)              bytes and flops one pass cannot do without
  exact(case, seed)       the outputs in 64 bits
"""
from __future__ import annotations

import math

import torch

own = False

_TORCH = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16, "int32": torch.int32}
_NAME = {v: k for k, v in _TORCH.items()}
_SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}
_TYPESTR = {"float32": "<f4", "float16": "<f2", "bfloat16": "<u2", "int32": "<i4"}
_EPS = 1e-6


# ----------------------------------------------------------------------
# Cases
# ----------------------------------------------------------------------

def listed():
    return [
        # A decoding step of 32 sequences: the new token's queries and keys are
        # normed and rotated, its keys and values go into the cache.
        _norm_rope("norm_rope_decode_bf16", "bfloat16", "cached", 32, 1, 32, 8, 128, 128, "rms", False, S=2048),
        # The DiT's sequence: 17776 tokens, 30 heads of 64, layer norm,
        # neighbouring columns rotated.
        _norm_rope("norm_rope_prompt_bf16", "bfloat16", "packed", 1, 17776, 30, 30, 64, 64, "layer", True),
        # A training step's backward pass: two sequences of 4096 tokens, four
        # query heads to a key head.
        _norm_rope("norm_rope_backward_bf16", "bfloat16", "backward", 2, 4096, 32, 8, 128, 128, "rms", False),
        # A training step's forward pass over long sequences (out and the
        # rows' log-sums).
        _window("window_train_bf16", "bfloat16", "train", 1, 8192, 32, 8, 128, 4096, 4),
        # A padded batch of prompts of sizes nobody rounded.
        _window("window_ragged_fp16", "float16", "forward", 3, 777, 6, 2, 72, 100, 3, lengths=True),
        # The backward pass of a training step.
        _window("window_backward_bf16", "bfloat16", "backward", 2, 4096, 16, 4, 128, 1024, 4),
        # A decoding step of 16 sequences over caches of up to 8192 tokens.
        _window("window_decode_bf16", "bfloat16", "cached", 16, 1, 32, 8, 128, 4096, 4, S=8192),
        # One long conversation, every token of the cache visible.
        _window("window_decode_long_fp16", "float16", "cached", 1, 1, 32, 8, 128, 0, 0, S=131072),
        # One token through the up-projections of a transformer MLP: decoding,
        # bound by reading the weights.
        _gated("gated_decode_bf16", "bfloat16", "forward", 1, 4096, 11008, "silu", False),
        # 4096 tokens through the same layer, with what its backward pass needs.
        _gated("gated_train_bf16", "bfloat16", "train", 4096, 4096, 11008, "silu", False),
        # Odd feature counts, a few hundred rows, biases.
        _gated("gated_ragged_fp16", "float16", "forward", 333, 1001, 1283, "gelu", True),
        # The backward pass at the DiT's widths.
        _gated("gated_backward_bf16", "bfloat16", "backward", 4096, 1920, 7680, "gelu", True),
    ]


def _norm_rope(name, dtype, way, B, n, H, Hk, D, R, norm, pairs, S=0):
    """H query and Hk key heads of D columns, the first R of them rotated;
    pairs: neighbouring columns, or the halves of R."""
    return {"name": name, "op": "norm_rope", "way": way, "dtype": dtype, "B": B, "n": n, "H": H, "Hk": Hk, "D": D,
            "R": R, "norm": norm, "pairs": pairs, "S": S}


def _window(name, dtype, way, B, n, H, Hk, D, window, sinks, S=0, lengths=False):
    """window 0: every key up to the query's own."""
    return {"name": name, "op": "window", "way": way, "dtype": dtype, "B": B, "n": n, "H": H, "Hk": Hk, "D": D,
            "window": window, "sinks": sinks, "S": S, "lengths": lengths}


def _gated(name, dtype, way, rows, K, F, act, bias):
    return {"name": name, "op": "gated", "way": way, "dtype": dtype, "rows": rows, "K": K, "F": F, "act": act,
            "bias": bias}


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _feature(rng, lo, hi):
    """A feature count: mostly a multiple of 64, at times of 8, at times odd."""
    n = _log(rng, lo, hi)
    kind = rng.random()
    if kind < 0.6:
        return max(64, n // 64 * 64)
    if kind < 0.8:
        return max(8, n // 8 * 8)
    return n | 1


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50.0)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        case = _draw_one(rng)
        # the plain attention holds every pair's score
        if case["op"] == "window" and case["way"] != "cached" and case["B"] * case["H"] * case["n"] ** 2 > 2 ** 31:
            continue
        if _cost(case) <= most:
            return case


def _draw_one(rng):
    op = rng.choice(("norm_rope", "window", "window", "gated"))
    half = rng.choice(("bfloat16", "float16"))
    Hk = _log(rng, 1, 16)
    H = Hk * rng.choice((1, 2, 3, 4, 8))
    if op == "norm_rope":
        way = rng.choice(("packed", "cached", "backward"))
        D = rng.choice((32, 64, 72, 80, 96, 128, 128, 256))
        cached = way == "cached"
        n = _log(rng, 1, 64) if cached else _log(rng, 1, 8192)
        return {"op": op, "way": way, "dtype": rng.choice((half, half, "float32")),
                "B": _log(rng, 1, 32) if cached else _log(rng, 1, 4), "n": n, "H": H, "Hk": Hk, "D": D,
                "R": rng.choice((D, D, D // 2)), "norm": rng.choice(("rms", "rms", "layer")),
                "pairs": rng.random() < 0.3, "S": n + _log(rng, 1, 2048) if cached else 0}
    if op == "window":
        way = rng.choice(("forward", "train", "backward", "cached", "cached"))
        cached = way == "cached"
        n = rng.choice((1, 1, 1, _log(rng, 2, 300))) if cached else _log(rng, 1, 8192)
        return {"op": op, "way": way, "dtype": half, "B": _log(rng, 1, 16) if cached else _log(rng, 1, 4), "n": n,
                "H": H, "Hk": Hk, "D": rng.choice((32, 64, 72, 96, 128, 128)),
                "window": rng.choice((0, _log(rng, 16, 4096), _log(rng, 16, 4096))),
                "sinks": rng.choice((0, 1, 4, 4, rng.randint(2, 100))),
                "S": n + _log(rng, 16, 32768) if cached else 0,
                "lengths": way in ("forward", "backward") and rng.random() < 0.5}
    way = rng.choice(("forward", "train", "backward"))
    return {"op": op, "way": way, "dtype": rng.choice((half, half, half, "float32")), "rows": _log(rng, 1, 8192),
            "K": _feature(rng, 64, 8192), "F": _feature(rng, 64, 11008), "act": rng.choice(("silu", "gelu")),
            "bias": rng.random() < 0.5}


# ----------------------------------------------------------------------
# Inputs
# ----------------------------------------------------------------------

def _inputs(case, seed):
    """The case's inputs as torch tensors, in a fixed order of draws."""
    c, dt = case, _TORCH[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    host = torch.Generator().manual_seed(int(seed))

    def normal(shape, std=1.0):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(dt)

    def counts(lo, hi):
        """One sequence of the longest, the others anywhere."""
        n = torch.randint(lo, hi + 1, (c["B"],), generator=host)
        n[int(torch.randint(0, c["B"], (1,), generator=host))] = hi
        return n.to(torch.int32).cuda()

    op = c["op"]
    if op == "gated":
        M, K, F = c["rows"], c["K"], c["F"]
        t = {"x": normal((M, K)), "w": normal((2 * F, K), 0.02)}
        if c["way"] == "backward":
            t["pre"] = normal((M, 2 * F))
            t["g"] = normal((M, F), 0.1)
        elif c["bias"]:
            t["b"] = normal((2 * F,), 0.01)
        return t
    B, n, H, Hk, D, S = (c[k] for k in ("B", "n", "H", "Hk", "D", "S"))
    t = {}
    if c["way"] == "cached":
        t["k"], t["v"] = normal((B, S, Hk * D)), normal((B, S, Hk * D))
        t["lengths"] = counts((S - n) // 2, S - n)
    elif c.get("lengths"):
        t["lengths"] = counts((n + 1) // 2, n)
    if op == "norm_rope":
        # columns differ in spread, as a projection's do
        spread = torch.rand((H + 2 * Hk) * D, generator=g, device="cuda").add_(0.5)
        t["x"] = (torch.randn((B, n, (H + 2 * Hk) * D), generator=g, device="cuda") * spread).to(dt)
        t["weight"] = (torch.rand((2, D), generator=g, device="cuda").add_(0.5)).to(dt)
        if c["norm"] == "layer":
            t["bias"] = normal((2, D), 0.1)
        at = torch.arange(max(S, n), dtype=torch.float64)
        turn = at[:, None] * 10000.0 ** (-torch.arange(0, c["R"], 2, dtype=torch.float64) / c["R"])
        t["table"] = torch.cat([turn.cos(), turn.sin()], 1).float().cuda()
        if c["way"] == "backward":
            t["g"] = normal((B, n, (H + 2 * Hk) * D), 0.1)
        return t
    if c["way"] == "cached":
        t["q"] = normal((B, n, H * D))
        return t
    t["x"] = normal((B, n, (H + 2 * Hk) * D))
    if c["way"] == "backward":
        t["g"] = normal((B, n, H * D), 0.1)
    return t


class _Memory:
    """A framework buffer as torch reads it (the array interface)."""

    __slots__ = ("__cuda_array_interface__", "keep")

    def __init__(self, gt, dtype):
        self.keep = gt
        self.__cuda_array_interface__ = {"shape": gt.shape, "typestr": _TYPESTR[dtype],
                                         "data": (gt.data_ptr, False), "version": 2}


def _view(t):
    """A torch tensor over a framework tensor's memory, which it keeps alive."""
    dtype = t.dtype.value
    v = torch.as_tensor(_Memory(t._gpu, dtype), device="cuda")
    return v.view(torch.bfloat16) if dtype == "bfloat16" else v


def _to_sf(t):
    """A framework tensor with the values and the layout of a torch one."""
    import scaffolding_amd as sf

    out = sf.empty(*t.shape, dtype=_NAME[t.dtype], device="cuda")
    _view(out).copy_(t)
    return out


def prepare(case, seed):
    c, t = case, _inputs(case, seed)
    if c["op"] == "window" and c["way"] == "backward":
        # what the forward pass left: its output and the rows' log-sums
        out, lse = _attention(c, *_heads(c, t["x"]), _seen(c, t))
        t["out"], t["lse"] = out.to(t["x"].dtype), lse.contiguous()
    if own:  # the same values in the framework's own buffers
        t = {n: _to_sf(v) for n, v in t.items()}
    return {"case": dict(case), "t": t}


# ----------------------------------------------------------------------
# One pass
# ----------------------------------------------------------------------

def run(state):
    c, t = state["case"], state["t"]
    if own:
        return _run_own(c, t)
    return {"norm_rope": _plain_norm_rope, "window": _plain_window, "gated": _plain_gated}[c["op"]](c, t)


def _run_own(c, t):
    from scaffolding_amd.nn import functional as F

    op, way = c["op"], c["way"]
    if op == "gated":
        if way == "backward":
            dx, dw, db = F.gated_linear_backward(t["g"], t["x"], t["w"], t["pre"], c["bias"], c["act"])
            return {"dx": _view(dx), "dw": _view(dw), **({"db": _view(db)} if c["bias"] else {})}
        if way == "train":
            y, pre = F.gated_linear(t["x"], t["w"], t.get("b"), c["act"], return_pre=True)
            return {"y": _view(y), "pre": _view(pre)}
        return _view(F.gated_linear(t["x"], t["w"], t.get("b"), c["act"]))
    if op == "norm_rope":
        how = dict(weight=t["weight"], norm=c["norm"], eps=_EPS, interleaved=c["pairs"])
        if way == "backward":
            dx, dw, db = F.qk_norm_rope_backward(t["g"], t["x"], c["H"], c["Hk"], t["table"], **how)
            return {"dx": _view(dx), "dw": _view(dw), **({"db": _view(db)} if c["norm"] == "layer" else {})}
        if way == "cached":
            q = F.qk_norm_rope_cached(t["x"], c["H"], c["Hk"], t["table"], t["k"], t["v"], t["lengths"],
                                      bias=t.get("bias"), **how)
            return {"q": _view(q), "k": _view(t["k"]), "v": _view(t["v"])}
        return _view(F.qk_norm_rope(t["x"], c["H"], c["Hk"], t["table"], bias=t.get("bias"), **how))
    window = c["window"] or None
    if way == "cached":
        return _view(F.window_attention_cached(t["q"], t["k"], t["v"], t["lengths"], c["H"], c["Hk"], window,
                                               c["sinks"]))
    if way == "backward":
        return _view(F.window_attention_backward(t["g"], t["x"], t["out"], t["lse"], c["H"], c["Hk"], window,
                                                 c["sinks"], lengths=t.get("lengths")))
    if way == "train":
        out, lse = F.window_attention(t["x"], c["H"], c["Hk"], window, c["sinks"], return_lse=True)
        return {"out": _view(out), "lse": _view(lse)}
    return _view(F.window_attention(t["x"], c["H"], c["Hk"], window, c["sinks"], lengths=t.get("lengths")))


def _act(y, act):
    if act == "silu":
        return y / (1.0 + torch.exp(-y))
    return 0.5 * y * (1.0 + torch.tanh(0.7978845608 * (y + 0.044715 * y * y * y)))


def _act_slope(x, act):
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-x))
        return s * (1.0 + x * (1.0 - s))
    u = torch.tanh(0.7978845608 * (x + 0.044715 * x * x * x))
    return 0.5 * (1.0 + u) + 0.5 * x * (1.0 - u * u) * 0.7978845608 * (1.0 + 3.0 * 0.044715 * x * x)


def _plain_gated(c, t):
    dt, F = _TORCH[c["dtype"]], c["F"]
    x, w = t["x"].float(), t["w"].float()
    if c["way"] != "backward":
        pre = x @ w.t()
        if c["bias"]:
            pre = pre + t["b"].float()
        y = (_act(pre[:, :F], c["act"]) * pre[:, F:]).to(dt)
        return {"y": y, "pre": pre.to(dt)} if c["way"] == "train" else y
    g, gate, up = t["g"].float(), t["pre"][:, :F].float(), t["pre"][:, F:].float()
    d = torch.cat([g * up * _act_slope(gate, c["act"]), g * _act(gate, c["act"])], 1)
    out = {"dx": (d @ w).to(dt), "dw": (d.t() @ x).to(dt)}
    if c["bias"]:
        out["db"] = d.sum(0).to(dt)
    return out


def _columns(c):
    """The two columns of each rotated pair."""
    R = c["R"]
    a = torch.arange(0, R, 2, device="cuda") if c["pairs"] else torch.arange(R // 2, device="cuda")
    return (a, a + 1) if c["pairs"] else (a, a + R // 2)


def _turns(c, t):
    """cos and sin, (B or 1, n, 1, R / 2)."""
    at = torch.arange(c["n"], device="cuda")[None]
    if c["way"] == "cached":
        at = at + t["lengths"][:, None]
    turn = t["table"][at][:, :, None]
    return turn[..., :c["R"] // 2], turn[..., c["R"] // 2:]


def _rotate(c, y, cos, sin):
    i, j = _columns(c)
    a, b = y[..., i], y[..., j]
    out = y.clone()
    out[..., i], out[..., j] = a * cos - b * sin, b * cos + a * sin
    return out


def _normed(c, x):
    """x / its norm over the head's columns, and 1 / that norm."""
    if c["norm"] == "layer":
        x = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
    return x * r, r


def _per_head(c, t, name):
    """The queries' row of a (2, D) parameter for each query head, the keys'
    for each key head."""
    p = t[name].float()
    return torch.cat([p[:1].expand(c["H"], -1), p[1:].expand(c["Hk"], -1)])


def _plain_norm_rope(c, t):
    dt, B, n, H, Hk, D = t["x"].dtype, c["B"], c["n"], c["H"], c["Hk"], c["D"]
    x = t["x"].view(B, n, H + 2 * Hk, D)
    hat, r = _normed(c, x[:, :, :H + Hk].float())
    w = _per_head(c, t, "weight")
    cos, sin = _turns(c, t)
    if c["way"] == "backward":
        g = t["g"].view(B, n, H + 2 * Hk, D)
        d = _rotate(c, g[:, :, :H + Hk].float(), cos, -sin)
        dw, db = (d * hat).sum((0, 1)), d.sum((0, 1))
        d = d * w
        back = d - hat * (d * hat).mean(-1, keepdim=True)
        if c["norm"] == "layer":
            back = back - d.mean(-1, keepdim=True)
        dx = torch.cat([(back * r).to(dt), g[:, :, H + Hk:]], 2).view_as(t["x"])
        out = {"dx": dx, "dw": torch.stack([dw[:H].sum(0), dw[H:].sum(0)]).to(dt)}
        if c["norm"] == "layer":
            out["db"] = torch.stack([db[:H].sum(0), db[H:].sum(0)]).to(dt)
        return out
    y = hat * w
    if c["norm"] == "layer":
        y = y + _per_head(c, t, "bias")
    y = _rotate(c, y, cos, sin).to(dt)
    if c["way"] == "packed":
        return torch.cat([y, x[:, :, H + Hk:]], 2).view_as(t["x"])
    at = t["lengths"][:, None].long() + torch.arange(n, device="cuda")
    b = torch.arange(B, device="cuda")[:, None]
    t["k"][b, at] = y[:, :, H:].reshape(B, n, Hk * D)
    t["v"][b, at] = x[:, :, H + Hk:].reshape(B, n, Hk * D)
    return {"q": y[:, :, :H].reshape(B, n, H * D), "k": t["k"], "v": t["v"]}


def _heads(c, x):
    """Queries (B, Hk, H / Hk, n, D), keys and values (B, Hk, 1, n, D) of a
    packed projection, fp32."""
    B, n, H, Hk, D = c["B"], c["n"], c["H"], c["Hk"], c["D"]
    x = x.view(B, n, H + 2 * Hk, D).float().transpose(1, 2).contiguous()
    return x[:, :H].view(B, Hk, H // Hk, n, D), x[:, H:H + Hk, None], x[:, H + Hk:, None]


def _seen(c, t):
    """Which keys each query sees, (B or 1, 1, 1, queries, keys)."""
    n = c["n"]
    keys = torch.arange(c["S"] if c["way"] == "cached" else n, device="cuda")
    at = torch.arange(n, device="cuda")[None]
    if c["way"] == "cached":
        at = at + t["lengths"][:, None]
    at = at[..., None]
    ok = keys <= at
    if c["window"]:
        ok = ok & ((keys > at - c["window"]) | (keys < c["sinks"]))
    if c["way"] != "cached" and c["lengths"]:
        ends = t["lengths"][:, None, None]
        ok = ok & (keys < ends) & (at < ends)
    return ok[:, None, None]


def _weights(c, q, k, ok):
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(c["D"])
    s = s.masked_fill_(~ok, -math.inf)
    most = s.amax(-1, keepdim=True)
    none = most == -math.inf  # no key at all: 0
    most = most.masked_fill(none, 0.0)
    p = torch.exp(s.sub_(most))
    total = p.sum(-1, keepdim=True)
    return p.div_(total.masked_fill(none, 1.0)), (most + torch.log(total))[..., 0]


def _attention(c, q, k, v, ok):
    """The output (B, n, H D) and the rows' log-sums (B, H, n), fp32."""
    p, lse = _weights(c, q, k, ok)
    out = torch.matmul(p, v).reshape(c["B"], c["H"], c["n"], c["D"])
    return out.transpose(1, 2).reshape(c["B"], c["n"], c["H"] * c["D"]), lse.reshape(c["B"], c["H"], c["n"])


def _plain_window(c, t):
    dt, B, n, H, Hk, D = _TORCH[c["dtype"]], c["B"], c["n"], c["H"], c["Hk"], c["D"]
    ok = _seen(c, t)
    if c["way"] == "cached":
        q = t["q"].view(B, n, Hk, H // Hk, D).float().permute(0, 2, 3, 1, 4).contiguous()
        k, v = (t[a].view(B, -1, Hk, 1, D).permute(0, 2, 3, 1, 4).float().contiguous() for a in ("k", "v"))
        return _attention(c, q, k, v, ok)[0].to(dt)
    q, k, v = _heads(c, t["x"])
    if c["way"] != "backward":
        out, lse = _attention(c, q, k, v, ok)
        return {"out": out.to(dt), "lse": lse} if c["way"] == "train" else out.to(dt)
    p, _ = _weights(c, q, k, ok)
    g = t["g"].view(B, n, H, D).float().transpose(1, 2).reshape(B, Hk, H // Hk, n, D)
    dv = torch.matmul(p.transpose(-1, -2).contiguous(), g).sum(2)
    dp = torch.matmul(g, v.transpose(-1, -2).contiguous())
    ds = dp.sub_((dp * p).sum(-1, keepdim=True)).mul_(p).div_(math.sqrt(D))
    dq = torch.matmul(ds, k).reshape(B, H, n, D)
    dk = torch.matmul(ds.transpose(-1, -2).contiguous(), q).sum(2)
    return torch.cat([dq, dk, dv], 1).transpose(1, 2).reshape(B, n, (H + 2 * Hk) * D).to(dt)


# ----------------------------------------------------------------------
# Work and 64-bit outputs
# ----------------------------------------------------------------------

def _visible(first, last, window, sinks):
    """Keys seen by the queries at positions first .. last - 1 (key and query
    pairs), and keys that any of them sees."""
    at = torch.arange(first, last, dtype=torch.float64)
    near = (at + 1).clamp(max=float(window or last))
    far = (at + 1 - near).clamp(max=float(sinks))
    keys = min(last, (window or last) + last - first - 1)
    return float((near + far).sum()), keys + min(sinks, last - keys)


def work(case):
    c, e = case, _SIZE[case["dtype"]]
    op, way = c["op"], c["way"]
    if op == "gated":
        M, K, F = c["rows"], c["K"], c["F"]
        if way == "backward":  # x, pre, g and w read, dx, dw and db written
            return {"bytes": e * (2 * M * K + 4 * F * K + 3 * M * F + (2 * F if c["bias"] else 0)),
                    "flops": 8.0 * M * K * F}
        b = e * (M * K + 2 * F * K + M * F + (2 * F if c["bias"] else 0) + (2 * M * F if way == "train" else 0))
        return {"bytes": b, "flops": 4.0 * M * K * F}
    B, n, H, Hk, D = (c[k] for k in ("B", "n", "H", "Hk", "D"))
    if op == "norm_rope":
        # read and written once; the gradient reads its operand's queries and keys too
        b = 2 * e * B * n * (H + 2 * Hk) * D + 2 * e * D
        b += 2 * c["R"] * (B * n * 2 if way == "cached" else 2 * n)
        if way == "backward":
            b += e * B * n * (H + Hk) * D
        return {"bytes": b, "flops": (12.0 if way == "backward" else 7.0) * B * n * (H + Hk) * D}
    if way == "cached":
        last = n + (c["S"] - n if B == 1 else (c["S"] - n) * 3 // 4)  # in the mean
        pairs, keys = _visible(last - n, last, c["window"], c["sinks"])
        return {"bytes": e * B * D * (2 * n * H + 2 * keys * Hk), "flops": 4.0 * B * H * D * pairs}
    last = n * 3 // 4 if c["lengths"] and B > 1 else n
    pairs, _ = _visible(0, last, c["window"], c["sinks"])
    tokens = B * n * D * (2 * H + 2 * Hk)  # queries, keys, values and the output
    if way == "backward":  # those and the gradient read, three gradients written
        return {"bytes": e * (tokens + B * n * D * (2 * H + 2 * Hk)) + 4 * B * H * n, "flops": 10.0 * B * H * D * pairs}
    return {"bytes": e * tokens + (4 * B * H * n if way == "train" else 0), "flops": 4.0 * B * H * D * pairs}


def exact(case, seed):
    c, t = case, _inputs(case, seed)
    return {"norm_rope": _exact_norm_rope, "window": _exact_window, "gated": _exact_gated}[c["op"]](c, t)


def _exact_act(y, act):
    if act == "silu":
        return y * torch.sigmoid(y)
    return torch.nn.functional.gelu(y, approximate="tanh")


def _exact_gated(c, t):
    x, w, F = t["x"].double(), t["w"].double(), c["F"]
    if c["way"] == "backward":
        pre = t["pre"].double().requires_grad_(True)
        y = _exact_act(pre[:, :F], c["act"]) * pre[:, F:]
        (d,) = torch.autograd.grad(y, pre, t["g"].double())
        out = {"dx": d @ w, "dw": d.T @ x}
        if c["bias"]:
            out["db"] = d.sum(0)
        return out
    gate, up = x @ w[:F].T, x @ w[F:].T
    if c["bias"]:
        gate, up = gate + t["b"][:F].double(), up + t["b"][F:].double()
    y = _exact_act(gate, c["act"]) * up
    return {"y": y, "pre": torch.cat([gate, up], 1)} if c["way"] == "train" else y


def _exact_norm_rope(c, t):
    B, n, H, Hk, D, R = (c[k] for k in ("B", "n", "H", "Hk", "D", "R"))
    x = t["x"].double().view(B, n, H + 2 * Hk, D)
    qk = x[:, :, :H + Hk].clone().requires_grad_(True)
    w = t["weight"].double().requires_grad_(True)
    b = t["bias"].double() if c["norm"] == "layer" else torch.zeros_like(w)
    b = b.detach().requires_grad_(True)
    of = torch.tensor([0] * H + [1] * Hk, device="cuda")
    y = qk - qk.mean(-1, keepdim=True) if c["norm"] == "layer" else qk
    y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + _EPS) * w[of] + b[of]
    # each rotated pair as one complex number, times e^(i angle)
    at = torch.arange(n, device="cuda").expand(B, n)
    if c["way"] == "cached":
        at = at + t["lengths"][:, None].long()
    tab = t["table"].double()[at]
    turn = torch.complex(tab[..., :R // 2], tab[..., R // 2:])[:, :, None]
    pair = y[..., :R].unflatten(-1, (R // 2, 2)) if c["pairs"] else y[..., :R].unflatten(-1, (2, R // 2)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
    z = z.flatten(-2) if c["pairs"] else z.transpose(-1, -2).flatten(-2)
    y = torch.cat([z, y[..., R:]], -1)
    if c["way"] == "backward":
        g = t["g"].double().view(B, n, H + 2 * Hk, D)
        d, dw, db = torch.autograd.grad(y, (qk, w, b), g[:, :, :H + Hk].contiguous())
        out = {"dx": torch.cat([d, g[:, :, H + Hk:]], 2).flatten(2), "dw": dw}
        if c["norm"] == "layer":
            out["db"] = db
        return out
    y = y.detach()
    if c["way"] == "packed":
        return torch.cat([y, x[:, :, H + Hk:]], 2).flatten(2)
    k, v = t["k"].double(), t["v"].double()
    for i, m in enumerate(t["lengths"].tolist()):
        k[i, m:m + n] = y[i, :, H:].flatten(1)
        v[i, m:m + n] = x[i, :, H + Hk:].flatten(1)
    return {"q": y[:, :, :H].flatten(2), "k": k, "v": v}


def _exact_window(c, t):
    """One sequence and head at a time, each query's keys counted out."""
    B, n, H, Hk, D = (c[k] for k in ("B", "n", "H", "Hk", "D"))
    back = c["way"] == "backward"
    out = torch.zeros((B, n, (H + 2 * Hk if back else H), D), dtype=torch.float64, device="cuda")
    lse = torch.full((B, H, n), -math.inf, dtype=torch.float64, device="cuda")
    ends = t["lengths"].tolist() if "lengths" in t else [n] * B
    for b in range(B):
        if c["way"] == "cached":
            first, rows, keys = ends[b], n, ends[b] + n
        else:
            first, rows, keys = 0, ends[b], ends[b]
        ago = torch.arange(first, first + rows, device="cuda")[:, None] - torch.arange(keys, device="cuda")
        hidden = ago < 0
        if c["window"]:
            hidden = hidden | ((ago >= c["window"]) & (torch.arange(keys, device="cuda") >= c["sinks"]))
        for h in range(H):
            u = h // (H // Hk)
            if c["way"] == "cached":
                q, k, v = t["q"][b].view(n, H, D)[:, h], t["k"][b, :keys].view(keys, Hk, D)[:, u], t["v"][b, :keys].view(keys, Hk, D)[:, u]
            else:
                x = t["x"][b, :rows].view(rows, H + 2 * Hk, D)
                q, k, v = x[:, h], x[:, H + u], x[:, H + Hk + u]
            q, k, v = (a.double().requires_grad_(back) for a in (q, k, v))
            s = (q @ k.T / D ** 0.5).masked_fill(hidden, -math.inf)
            o = torch.softmax(s, 1) @ v
            if back:
                g = t["g"][b, :rows].view(rows, H, D)[:, h].double()
                dq, dk, dv = torch.autograd.grad(o, (q, k, v), g)
                out[b, :rows, h] = dq
                out[b, :rows, H + u] += dk
                out[b, :rows, H + Hk + u] += dv
            else:
                out[b, :rows, h] = o
                lse[b, h, :rows] = torch.logsumexp(s, 1)
    out = out.flatten(2)
    return {"out": out, "lse": lse} if c["way"] == "train" else out

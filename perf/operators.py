"""Performance cases of the expert operators and the 4-bit linear layer.

  route      top-k routing of tokens to experts, with its gradient
  rows       tokens to expert order and back (dispatch, combine, combine's
             gradient)
  grouped    a linear layer with one weight per expert over ragged groups of
             rows, and its backward pass
  q4         a linear layer with 4-bit weights and group scales, dense or one
             weight per expert

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

_TORCH = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16, "int32": torch.int32,
          "uint8": torch.uint8}
_NAME = {v: k for k, v in _TORCH.items()}
_SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}
_TYPESTR = {"float32": "<f4", "float16": "<f2", "bfloat16": "<u2", "int32": "<i4", "uint8": "|u1"}


# ----------------------------------------------------------------------
# Cases
# ----------------------------------------------------------------------

def listed():
    return [
        # A small fp32 expert layer (a test-sized model, a conditioning
        # embedding): launch and host time.
        _grouped("grouped_small_fp32", "float32", 64, 4, 512, 512, "none"),
        # Decoding: 8 tokens, two experts each, through the up-projection of a
        # transformer MLP; bound by reading the chosen experts' weights.
        _grouped("grouped_decode_bf16", "bfloat16", 16, 8, 4096, 11008, "silu"),
        # 4096 tokens, two experts each, at the DiT's widths: the ordinary
        # training or prompt pass.
        _grouped("grouped_large_bf16", "bfloat16", 8192, 8, 1920, 7680, "silu"),
        # Sizes nobody rounded: odd feature counts, more experts than a power
        # of two, groups of a few dozen rows.
        _grouped("grouped_ragged_fp16", "float16", 777, 13, 1001, 1283, "gelu"),
        # The backward pass of the up-projection with its activation: dX, dW
        # and the bias gradient of each expert.
        _grouped("grouped_backward_bf16", "bfloat16", 4096, 8, 1920, 7680, "silu", "backward"),
        # One token through a 4-bit up-projection: decoding.
        _q4("q4_decode_bf16", "bfloat16", 1, 1, 4096, 11008, 128, False, "silu"),
        # A batch of 13 sequences through a 4-bit down-projection with zero
        # points.
        _q4("q4_batch_fp16", "float16", 13, 1, 11008, 4096, 64, True, "none"),
        # Decoding through 4-bit experts: 8 tokens, two experts each.
        _q4("q4_experts_bf16", "bfloat16", 16, 8, 4096, 11008, 128, False, "silu"),
        # The router of a decoding step.
        _route("route_decode_fp32", "float32", 16, 8, 2, True, False, False),
        # The router of a training step over 16384 tokens, with its gradient.
        _route("route_train_bf16", "bfloat16", 16384, 64, 8, True, False, True),
        # The experts' answers for 4096 tokens, two each, summed per token.
        _rows("combine_bf16", "bfloat16", 4096, 2, 4096, "combine"),
        # Its backward pass, at a width that is no multiple of 8.
        _rows("combine_backward_fp16", "float16", 4096, 2, 1283, "combine_backward"),
    ]


def _grouped(name, dtype, rows, E, K, N, act, way="forward"):
    return {"name": name, "op": "grouped", "way": way, "dtype": dtype, "rows": rows, "E": E, "K": K, "N": N,
            "act": act}


def _q4(name, dtype, rows, E, K, N, group, zeros, act):
    return {"name": name, "op": "q4", "dtype": dtype, "rows": rows, "E": E, "K": K, "N": N, "group": group,
            "zeros": zeros, "act": act}


def _route(name, dtype, T, E, k, renorm, masked, train):
    return {"name": name, "op": "route", "dtype": dtype, "T": T, "E": E, "k": k, "renorm": renorm, "masked": masked,
            "train": train}


def _rows(name, dtype, T, k, D, way):
    return {"name": name, "op": "rows", "way": way, "dtype": dtype, "T": T, "k": k, "D": D}


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
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
        if _cost(case) <= most:
            return case


def _draw_one(rng):
    op = rng.choice(("grouped", "grouped", "grouped", "q4", "q4", "route", "rows"))
    half = rng.choice(("bfloat16", "float16"))
    if op == "grouped":
        way = rng.choice(("forward", "forward", "backward"))
        return {"op": op, "way": way, "dtype": rng.choice((half, half, half, "float32")),
                "rows": _log(rng, 1, 16384), "E": _log(rng, 1, 64), "K": _width(rng, 64, 11008),
                "N": _width(rng, 64, 11008), "act": rng.choice(("none", "silu", "gelu"))}
    if op == "q4":
        group = rng.choice((32, 64, 128))
        return {"op": op, "dtype": half, "rows": _log(rng, 1, 512), "E": rng.choice((1, 1, 1, _log(rng, 2, 16))),
                "K": max(1, _log(rng, 256, 11008) // group) * group, "N": _width(rng, 256, 11008), "group": group,
                "zeros": rng.random() < 0.5, "act": rng.choice(("none", "silu", "gelu"))}
    if op == "route":
        E = _log(rng, 2, 256)
        return {"op": op, "dtype": rng.choice((half, "float32")), "T": _log(rng, 1, 16384), "E": E,
                "k": rng.randint(1, min(E, 8)), "renorm": rng.random() < 0.5, "masked": rng.random() < 0.3,
                "train": rng.random() < 0.5}
    return {"op": op, "way": rng.choice(("dispatch", "combine", "combine_backward")),
            "dtype": rng.choice((half, half, "float32")), "T": _log(rng, 1, 8192), "k": rng.randint(1, 8),
            "D": _width(rng, 64, 8192)}


# ----------------------------------------------------------------------
# Inputs
# ----------------------------------------------------------------------

def _inputs(case, seed):
    """The case's inputs as torch tensors, in a fixed order of draws."""
    c, dt = case, _TORCH[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    host = torch.Generator().manual_seed(int(seed))

    def normal(shape, std=1.0, dtype=dt):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(dtype)

    def offsets():
        """Group starts as a router gives them: experts are not equally
        liked, and some may get no row at all."""
        like = torch.randn(c["E"], generator=host).mul_(0.5).exp_()
        each = torch.multinomial(like, c["rows"], replacement=True, generator=host).bincount(minlength=c["E"])
        return torch.cat([torch.zeros(1, dtype=torch.int64), each.cumsum(0)]).to(torch.int32).cuda()

    op = c["op"]
    if op == "grouped":
        R, E, K, N = c["rows"], c["E"], c["K"], c["N"]
        t = {"offsets": offsets(), "x": normal((R, K)), "w": normal((E, N, K), 0.02)}
        if c["way"] == "forward":
            t["b"] = normal((E, N), 0.01)
        else:
            t["g"] = normal((R, N), 0.1)
            if c["act"] != "none":
                t["pre"] = normal((R, N))
        return t
    if op == "q4":
        E, K, N, G = c["E"], c["K"], c["N"], c["group"]
        lead = (E,) if E > 1 else ()
        t = {"x": normal((c["rows"], K)),
             "q": torch.randint(0, 256, lead + (N, K // 2), generator=g, device="cuda", dtype=torch.uint8),
             "s": (torch.rand(lead + (K // G, N), generator=g, device="cuda").add_(0.5).mul_(0.004)).to(dt),
             "b": normal(lead + (N,), 0.01)}
        if c["zeros"]:
            t["z"] = torch.randint(5, 12, lead + (K // G, N), generator=g, device="cuda", dtype=torch.uint8)
        if E > 1:
            t["offsets"] = offsets()
        return t
    if op == "route":
        T, E = c["T"], c["E"]
        v = torch.randn((T, E), generator=g, device="cuda").mul_(1.5)
        v += torch.randn((1, E), generator=g, device="cuda").mul_(0.5)
        if c["masked"]:  # experts a token may not use; now and then it may use none
            v.masked_fill_(torch.rand((T, E), generator=g, device="cuda") < 0.5, -math.inf)
            v.masked_fill_(torch.rand((T, 1), generator=g, device="cuda") < 0.05, -math.inf)
        t = {"logits": v.to(dt)}
        if c["train"]:
            t["g"] = normal((T, c["k"]), 0.1, torch.float32)
        return t
    T, k, D = c["T"], c["k"], c["D"]
    t = {"slots": torch.randperm(T * k, generator=host).to(torch.int32).reshape(T, k).cuda()}
    if c["way"] == "dispatch":
        t["x"] = normal((T, D))
        return t
    t["y"] = normal((T * k, D))
    w = torch.rand((T, k), generator=g, device="cuda").add_(0.1)
    t["w"] = w / w.sum(1, keepdim=True)
    if c["way"] == "combine_backward":
        t["g"] = normal((T, D), 0.1)
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
    t = _inputs(case, seed)
    # The rows of the largest group, which the plain form pads every group to:
    # a program that pads knows its capacity.
    cap = int((t["offsets"][1:] - t["offsets"][:-1]).max()) if "offsets" in t else 0
    if own:  # the same values in the framework's own buffers
        t = {n: _to_sf(v) for n, v in t.items()}
    return {"case": dict(case), "cap": cap, "t": t}


# ----------------------------------------------------------------------
# One pass
# ----------------------------------------------------------------------

def run(state):
    c, t = state["case"], state["t"]
    if own:
        return _run_own(c, t)
    op = c["op"]
    if op == "grouped":
        return _plain_grouped(c, t, state["cap"])
    if op == "q4":
        return _plain_q4(c, t, state["cap"])
    if op == "route":
        return _plain_route(c, t)
    return _plain_rows(c, t)


def _run_own(c, t):
    from scaffolding_amd.nn import functional as F

    op = c["op"]
    act = None if c.get("act") == "none" else c.get("act")
    if op == "grouped":
        if c["way"] == "forward":
            return _view(F.grouped_linear(t["x"], t["w"], t["offsets"], t["b"], act))
        dx, dw, db = F.grouped_linear_backward(t["g"], t["x"], t["w"], t["offsets"], True, act, t.get("pre"))
        return {"dx": _view(dx), "dw": _view(dw), "db": _view(db)}
    if op == "q4":
        return _view(F.linear_q4(t["x"], t["q"], t["s"], t.get("z"), t["b"], act, t.get("offsets")))
    if op == "route":
        r = F.route_topk(t["logits"], c["k"], c["renorm"])
        out = {"weights": _view(r.weights), "experts": _view(r.experts), "offsets": _view(r.offsets),
               "slots": _view(r.slots)}
        if c["train"]:
            out["dlogits"] = _view(F.route_topk_backward(t["g"], t["logits"], r))
        return out
    if c["way"] == "dispatch":
        return _view(F.dispatch_rows(t["x"], t["slots"]))
    if c["way"] == "combine":
        return _view(F.combine_rows(t["y"], t["slots"], t["w"]))
    dy, dw = F.combine_rows_backward(t["g"], t["y"], t["slots"], t["w"])
    return {"dy": _view(dy), "dw": _view(dw)}


def _act(y, act):
    if act == "silu":
        return y / (1.0 + torch.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1.0 + torch.tanh(0.7978845608 * (y + 0.044715 * y * y * y)))
    return y


def _act_slope(x, act):
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-x))
        return s * (1.0 + x * (1.0 - s))
    u = torch.tanh(0.7978845608 * (x + 0.044715 * x * x * x))
    return 0.5 * (1.0 + u) + 0.5 * x * (1.0 - u * u) * 0.7978845608 * (1.0 + 3.0 * 0.044715 * x * x)


def _places(offsets, rows):
    """Each row's group, and its place within it."""
    r = torch.arange(rows, device=offsets.device, dtype=torch.int32)
    e = torch.searchsorted(offsets[1:].contiguous(), r, right=True)
    return e, (r - offsets[e]).long()


def _padded(v, e, at, E, cap):
    p = torch.zeros((E, cap, v.shape[1]), device=v.device)
    p[e, at] = v.float()
    return p


def _products(x, w, b, e, at, E, cap):
    """x[r] . w[e[r]]^T + b[e[r]]: the weight on the left, as it lies."""
    y = torch.bmm(w, _padded(x, e, at, E, cap).transpose(1, 2).contiguous()) + b.float()[:, :, None]
    return y[e, :, at]


def _plain_grouped(c, t, cap):
    dt, E = _TORCH[c["dtype"]], c["E"]
    e, at = _places(t["offsets"], c["rows"])
    w = t["w"].float()
    if c["way"] == "forward":
        return _act(_products(t["x"], w, t["b"], e, at, E, cap), c["act"]).to(dt)
    g = t["g"].float()
    if c["act"] != "none":
        g = g * _act_slope(t["pre"].float(), c["act"])
    g = _padded(g, e, at, E, cap)
    x = _padded(t["x"], e, at, E, cap)
    return {"dx": torch.bmm(g, w)[e, at].to(dt), "dw": torch.bmm(g.transpose(1, 2).contiguous(), x).to(dt),
            "db": g.sum(1).to(dt)}


def _plain_q4(c, t, cap):
    dt, G = _TORCH[c["dtype"]], c["group"]
    q = torch.stack([t["q"] & 15, t["q"] >> 4], -1).flatten(-2).float()
    q = q.unflatten(-1, (c["K"] // G, G))
    z = t["z"].float().transpose(-1, -2)[..., None] if c["zeros"] else 8.0
    w = ((q - z) * t["s"].float().transpose(-1, -2)[..., None]).flatten(-2)
    x, b = t["x"].float(), t["b"].float()
    if c["E"] == 1:
        return _act((w @ x.t().contiguous()).t() + b, c["act"]).to(dt)
    e, at = _places(t["offsets"], c["rows"])
    return _act(_products(x, w, b, e, at, c["E"], cap), c["act"]).to(dt)


def _plain_route(c, t):
    v, k = t["logits"].float(), c["k"]
    T, E = v.shape
    top, chosen = torch.sort(v, dim=1, descending=True, stable=True)
    top, chosen = top[:, :k], chosen[:, :k]
    most = top[:, :1]
    none = most == -math.inf  # no expert allowed: no weight for any
    most = torch.where(none, torch.zeros_like(most), most)
    p = torch.exp(v - most)
    w = torch.exp(top - most)
    total = (w if c["renorm"] else p).sum(1, keepdim=True)
    total = torch.where(none, torch.ones_like(total), total)
    w = w / total
    flat = chosen.reshape(-1)
    order = torch.sort(flat, dim=0, stable=True)[1]
    slots = torch.empty_like(order)
    slots[order] = torch.arange(T * k, device=v.device)
    each = (flat[None, :] == torch.arange(E, device=v.device)[:, None]).sum(1)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device=v.device), each.cumsum(0)])
    out = {"weights": w, "experts": chosen.to(torch.int32), "offsets": offsets.to(torch.int32),
           "slots": slots.to(torch.int32).reshape(T, k)}
    if c["train"]:
        g = t["g"]
        back = torch.zeros_like(v).scatter_(1, chosen, w * g)
        p = torch.zeros_like(v).scatter_(1, chosen, w) if c["renorm"] else p / total
        out["dlogits"] = (back - p * (w * g).sum(1, keepdim=True)).to(t["logits"].dtype)
    return out


def _plain_rows(c, t):
    dt, k = _TORCH[c["dtype"]], c["k"]
    at = t["slots"].long()
    if c["way"] == "dispatch":
        out = torch.empty((c["T"] * k, c["D"]), dtype=dt, device="cuda")
        out[at.reshape(-1)] = t["x"].repeat_interleave(k, 0)
        return out
    y = t["y"].float()[at]
    if c["way"] == "combine":
        return (y * t["w"][:, :, None]).sum(1).to(dt)
    g = t["g"].float()[:, None, :]
    dy = torch.empty_like(t["y"])
    dy[at.reshape(-1)] = (g * t["w"][:, :, None]).to(dt).reshape(-1, c["D"])
    return {"dy": dy, "dw": (g * y).sum(2)}


# ----------------------------------------------------------------------
# Work and 64-bit outputs
# ----------------------------------------------------------------------

def _reached(rows, E):
    """Experts with a row at all, in the mean of equally liked ones."""
    return E * (1.0 - (1.0 - 1.0 / E) ** rows)


def work(case):
    c, e = case, _SIZE[case["dtype"]]
    op = c["op"]
    if op == "grouped":
        R, E, K, N = c["rows"], c["E"], c["K"], c["N"]
        w = _reached(R, E)
        if c["way"] == "forward":
            return {"bytes": e * (R * K + w * N * K + w * N + R * N) + 4 * (E + 1), "flops": 2.0 * R * N * K}
        # the gradient of every expert's weight is written, of an empty one as zeros
        pre = R * N if c["act"] != "none" else 0
        return {"bytes": e * (R * N + pre + 2 * R * K + (w + E) * N * K + E * N) + 4 * (E + 1),
                "flops": 4.0 * R * N * K}
    if op == "q4":
        R, E, K, N = c["rows"], c["E"], c["K"], c["N"]
        w = _reached(R, E)
        per_group = e + (1 if c["zeros"] else 0)
        return {"bytes": w * (N * K / 2 + N * (K // c["group"]) * per_group + e * N) + e * R * (K + N),
                "flops": 2.0 * R * N * K}
    if op == "route":
        T, E, k = c["T"], c["E"], c["k"]
        back = 4 * T * k + e * T * E if c["train"] else 0
        return {"bytes": e * T * E + 12 * T * k + 4 * (E + 1) + back, "flops": 4.0 * T * E}
    T, k, D = c["T"], c["k"], c["D"]
    if c["way"] == "dispatch":
        return {"bytes": e * T * D * (k + 1) + 4 * T * k, "flops": 0.0}
    if c["way"] == "combine":
        return {"bytes": e * T * D * (k + 1) + 8 * T * k, "flops": 2.0 * T * k * D}
    return {"bytes": e * T * D * (2 * k + 1) + 12 * T * k, "flops": 3.0 * T * k * D}


def exact(case, seed):
    c = case
    t = _inputs(c, seed)
    op = c["op"]
    if op == "route":
        return _exact_route(c, t)
    if op == "rows":
        return _exact_rows(c, t)
    if op == "q4":
        low, high = (t["q"] % 16).double(), (t["q"] // 16).double()
        w = torch.zeros(t["q"].shape[:-1] + (c["K"],), dtype=torch.float64, device="cuda")
        w[..., 0::2], w[..., 1::2] = low, high
        of = torch.arange(c["K"], device="cuda") // c["group"]
        zero = t["z"].double() if c["zeros"] else torch.full(t["s"].shape, 8.0, device="cuda").double()
        w = (w - zero.transpose(-1, -2)[..., of]) * t["s"].double().transpose(-1, -2)[..., of]
        if c["E"] == 1:
            return _exact_act(t["x"].double() @ w.T + t["b"].double(), c["act"])
        t = {"x": t["x"], "w": w, "b": t["b"], "offsets": t["offsets"]}
    ends = t["offsets"].tolist()
    if op == "q4" or c["way"] == "forward":
        y = torch.zeros((c["rows"], c["N"]), dtype=torch.float64, device="cuda")
        for e in range(c["E"]):
            lo, hi = ends[e], ends[e + 1]
            y[lo:hi] = t["x"][lo:hi].double() @ t["w"][e].double().T + t["b"][e].double()
        return _exact_act(y, c["act"])
    g = t["g"].double()
    if c["act"] != "none":
        pre = t["pre"].double().requires_grad_(True)
        (slope,) = torch.autograd.grad(_exact_act(pre, c["act"]).sum(), pre)
        g = g * slope
    dx = torch.zeros((c["rows"], c["K"]), dtype=torch.float64, device="cuda")
    dw = torch.zeros((c["E"], c["N"], c["K"]), dtype=torch.float64, device="cuda")
    db = torch.zeros((c["E"], c["N"]), dtype=torch.float64, device="cuda")
    for e in range(c["E"]):
        lo, hi = ends[e], ends[e + 1]
        dx[lo:hi] = g[lo:hi] @ t["w"][e].double()
        dw[e] = g[lo:hi].T @ t["x"][lo:hi].double()
        db[e] = g[lo:hi].sum(0)
    return {"dx": dx, "dw": dw, "db": db}


def _exact_act(y, act):
    if act == "silu":
        return y * torch.sigmoid(y)
    if act == "gelu":
        return torch.nn.functional.gelu(y, approximate="tanh")
    return y


def _exact_route(c, t):
    import numpy as np

    v = t["logits"].double().cpu().numpy()
    T, E, k = c["T"], c["E"], c["k"]
    # the largest k logits; equal ones in the order of their index
    chosen = np.argsort(-v, axis=1, kind="stable")[:, :k]
    top = np.take_along_axis(v, chosen, 1)
    live = np.isfinite(top[:, :1])
    shift = np.where(live, top[:, :1], 0.0)
    p = np.where(live, np.exp(v - shift), 0.0)
    if c["renorm"]:
        held = np.zeros_like(p)
        np.put_along_axis(held, chosen, np.take_along_axis(p, chosen, 1), 1)
        p = held
    p = p / np.where(live, p.sum(1, keepdims=True), 1.0)
    w = np.take_along_axis(p, chosen, 1)
    flat = chosen.reshape(-1)
    slots = np.empty(T * k, np.int32)
    slots[np.argsort(flat, kind="stable")] = np.arange(T * k, dtype=np.int32)
    offsets = np.searchsorted(np.sort(flat), np.arange(E + 1)).astype(np.int32)
    out = {"weights": w, "experts": chosen.astype(np.int32), "offsets": offsets, "slots": slots.reshape(T, k)}
    if c["train"]:
        g = np.zeros_like(p)  # the softmax gradient: p (g - <p, g>)
        np.put_along_axis(g, chosen, t["g"].double().cpu().numpy(), 1)
        out["dlogits"] = p * (g - (p * g).sum(1, keepdims=True))
    return out


def _exact_rows(c, t):
    T, k, D = c["T"], c["k"], c["D"]
    slots = t["slots"].long()
    if c["way"] == "dispatch":
        out = torch.zeros((T * k, D), dtype=torch.float64, device="cuda")
        for j in range(k):
            out[slots[:, j]] = t["x"].double()
        return out
    y, w = t["y"].double(), t["w"].double()
    if c["way"] == "combine":
        out = torch.zeros((T, D), dtype=torch.float64, device="cuda")
        for j in range(k):
            out += w[:, j, None] * y[slots[:, j]]
        return out
    g = t["g"].double()
    dy = torch.zeros((T * k, D), dtype=torch.float64, device="cuda")
    dw = torch.zeros((T, k), dtype=torch.float64, device="cuda")
    for j in range(k):
        dy[slots[:, j]] = w[:, j, None] * g
        dw[:, j] = (g * y[slots[:, j]]).sum(1)
    return {"dy": dy, "dw": dw}

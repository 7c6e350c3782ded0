"""Performance cases of the dense operators beside the expert layer.

A model of mixture layers has dense parts next to them: the norm in front of
the router, layers whose feed-forward block is dense, an expert that every
token takes. Three operators, each in its plain form (elementary torch
operations in 32 bits, rounded once at the end) and as calls of
``triton_moe.kernels``:

- "norm": layer norm (``layer_norm``);
- "linear": a matrix product with bias, activation and residual in its
  epilogue (``fused_linear``): act(x w + b) + r;
- "gated": a gated feed-forward block (``gated_mlp``): h = act(x g + b_g) *
  (x u + b_u) with w1 = [g | u], and h w2 + b2 + r.

A "train" case is one forward and backward pass and returns the output and
every gradient. Weights are [in, out]; order "out_in" is the transposed view
of a matrix stored [out, in], as torch's Linear keeps it.
"""

from __future__ import annotations

import functools
import math
import os
import sys

import torch

own = False

GATES = {"swiglu": "silu", "geglu": "gelu", "geglu_tanh": "gelu_tanh", "reglu": "relu"}


def _norm(name, rows, d, dtype, train, weights="same"):
    """weights: "same" as the rows, "f32", or "none"."""
    return {"name": name, "kind": "norm", "rows": rows, "d": d, "dtype": dtype, "train": train,
            "weights": weights}


def _linear(name, rows, d, out, dtype, train, act, bias, residual, order="in_out"):
    return {"name": name, "kind": "linear", "rows": rows, "d": d, "out": out, "dtype": dtype,
            "train": train, "act": act, "bias": bias, "residual": residual, "order": order}


def _gated(name, rows, d, width, dtype, train, act, bias, residual, order="in_out"):
    return {"name": name, "kind": "gated", "rows": rows, "d": d, "width": width, "dtype": dtype,
            "train": train, "act": act, "bias": bias, "residual": residual, "order": order}


def listed():
    return [
        # the norm of one sequence generating alone: launch and latency
        _norm("norm_one_token", 1, 2048, "bf16", False),
        # a training step's tokens in front of a mixture layer, weights kept in
        # float32 beside bfloat16 rows
        _norm("norm_train", 32768, 2048, "bf16", True, "f32"),
        # a layer left in torch's default type, an odd number of tokens
        _norm("norm_train_f32", 4101, 768, "f32", True),
        # one token's projection back into the residual stream
        _linear("linear_one_token", 1, 2048, 2048, "bf16", False, "none", True, True),
        # a serving batch through the first layer of a plain block, with the
        # weight as torch's Linear stores it
        _linear("linear_batch", 61, 1024, 4096, "bf16", False, "gelu", True, False, "out_in"),
        # a prompt of odd length through a block's second layer
        _linear("linear_prefill", 4099, 4096, 2048, "bf16", False, "none", True, True),
        # a training step of a dense layer with the experts' activation
        _linear("linear_train", 8192, 1024, 4096, "bf16", True, "relu_squared", True, False),
        # the same in torch's default type, every operand of the epilogue
        _linear("linear_train_f32", 2051, 768, 2048, "f32", True, "gelu", True, True, "out_in"),
        # one token through the block that every token takes: its weights
        _gated("gated_one_token", 1, 2048, 5632, "bf16", False, "swiglu", False, True),
        # a serving batch, weights as torch's Linear stores them
        _gated("gated_batch", 23, 1024, 4096, "bf16", False, "swiglu", False, True, "out_in"),
        # a prompt
        _gated("gated_prefill", 4096, 2048, 8192, "bf16", False, "swiglu", False, True),
        # a training step of a large block
        _gated("gated_train", 16384, 2048, 8192, "bf16", True, "swiglu", False, True),
    ]


def _log_int(rng, lo, hi, mult=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / mult)) * mult))


def draw(rng):
    """One more case of the same ranges: 1 to 32768 rows, hidden sizes 64 to
    4096 and widths 64 to 8192 in steps of 8 (norms: 16 to 8192, any number),
    both types, with and without gradients. It costs no more than the largest
    listed case."""
    cost = lambda c: max(work(c)["bytes"] / 4e12, work(c)["flops"] / 1e14)  # noqa: E731
    limit = max(cost(c) for c in listed())
    while True:
        kind = rng.choice(["norm", "linear", "linear", "gated", "gated"])
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        train = rng.random() < 0.5
        rows = _log_int(rng, 1, 32768)
        if kind == "norm":
            c = _norm("", rows, _log_int(rng, 16, 8192), dtype, train,
                      rng.choice(["same", "same", "f32", "none"]))
        else:
            d, n = _log_int(rng, 64, 4096, 8), _log_int(rng, 64, 8192, 8)
            order = rng.choice(["in_out", "out_in"])
            flags = (rng.random() < 0.5, rng.random() < 0.5)
            if kind == "linear":
                act = rng.choice(["none", "none", "relu", "relu_squared", "silu", "gelu",
                                  "gelu_tanh"])
                c = _linear("", rows, d, n, dtype, train, act, *flags, order)
            else:
                c = _gated("", rows, d, n, dtype, train, rng.choice(sorted(GATES)), *flags, order)
        del c["name"]
        if cost(c) <= limit:
            return c


class _State:
    pass


@functools.lru_cache(None)
def _kernels():
    root = os.path.join(os.getcwd(), "triton-variable-moe_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from triton_moe import kernels
    return kernels


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * (seed % 100003) + 31)
    dtype = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
    train = case["train"]

    def normal(*shape, std=1.0, mean=0.0, dtype=dtype, leaf=True):
        t = torch.empty(*shape, device="cuda", dtype=torch.float32)
        return t.normal_(mean, std, generator=g).to(dtype).requires_grad_(leaf and train)

    def matrix(rows, cols):
        # in_out: as it is multiplied; out_in: a view of the stored transpose
        std = 1.0 / math.sqrt(rows)
        if case["order"] == "in_out":
            return normal(rows, cols, std=std)
        w = normal(cols, rows, std=std, leaf=False).t()
        return w.requires_grad_(train)

    s = _State()
    s.case = case
    rows, d = case["rows"], case["d"]
    s.x = s.w = s.b = s.w2 = s.b2 = s.r = s.gy = None
    if case["kind"] == "norm":
        # a residual stream: features of different scales, a few of them large
        scale = torch.exp(0.5 * normal(d, dtype=torch.float32, leaf=False))
        scale[:: max(1, d // 8)] *= 8.0
        x = normal(rows, d, dtype=torch.float32, leaf=False)
        s.x = (x * scale + 0.1 * scale).to(dtype).requires_grad_(train)
        if case["weights"] != "none":
            wt = torch.float32 if case["weights"] == "f32" else dtype
            s.w = normal(d, std=0.2, mean=1.0, dtype=wt)
            s.b = normal(d, std=0.2, dtype=wt)
        if train:
            s.gy = normal(rows, d, leaf=False)
        return s
    s.x = normal(rows, d)
    n = case["out"] if case["kind"] == "linear" else d
    if case["kind"] == "linear":
        s.w = matrix(d, n)
        s.b = normal(n, std=0.5) if case["bias"] else None
    else:
        s.w, s.w2 = matrix(d, 2 * case["width"]), matrix(case["width"], d)
        if case["bias"]:
            s.b, s.b2 = normal(2 * case["width"], std=0.5), normal(d, std=0.5)
    s.r = normal(rows, n) if case["residual"] else None
    if train:
        s.gy = normal(rows, n, leaf=False)
    return s


def _act(name, z):
    """The activation of z and its derivative."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return torch.clamp(z, min=0), (z > 0).to(z.dtype)
    if name == "relu_squared":
        p = torch.clamp(z, min=0)
        return p * p, 2 * p
    if name == "silu":
        t = 1 / (1 + torch.exp(-z))
        return z * t, t * (1 + z * (1 - t))
    if name == "gelu":
        phi = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z * z * z))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 0.134145 * z * z)


def _float(t):
    return None if t is None else t.detach().float()


def _plain_norm(s):
    x, w, b = _float(s.x), _float(s.w), _float(s.b)
    c = x - x.mean(dim=-1, keepdim=True)
    rstd = 1 / torch.sqrt((c * c).mean(dim=-1, keepdim=True) + 1e-5)
    n = c * rstd
    y = (n if w is None else n * w + b).to(s.x.dtype)
    if not s.case["train"]:
        return y
    gy = _float(s.gy)
    gn = gy if w is None else gy * w
    gx = rstd * (gn - gn.mean(dim=-1, keepdim=True) - n * (gn * n).mean(dim=-1, keepdim=True))
    out = [y, gx.to(s.x.dtype)]
    if w is not None:
        out += [(gy * n).sum(dim=0).to(s.w.dtype), gy.sum(dim=0).to(s.b.dtype)]
    return out


def _plain_linear(s):
    x, w, b, r = _float(s.x), _float(s.w), _float(s.b), _float(s.r)
    z = x @ w
    if b is not None:
        z = z + b
    y, slope = _act(s.case["act"], z)
    if r is not None:
        y = y + r
    y = y.to(s.x.dtype)
    if not s.case["train"]:
        return y
    gz = _float(s.gy) * slope
    out = [y, (gz @ w.t()).to(s.x.dtype), (x.t() @ gz).to(s.w.dtype)]
    if b is not None:
        out.append(gz.sum(dim=0).to(s.b.dtype))
    if r is not None:
        out.append(s.gy)
    return out


def _plain_gated(s):
    x, w1, w2, r = _float(s.x), _float(s.w), _float(s.w2), _float(s.r)
    z = x @ w1
    if s.b is not None:
        z = z + _float(s.b)
    gate, up = z.chunk(2, dim=1)
    a, slope = _act(GATES[s.case["act"]], gate)
    h = a * up
    y = h @ w2
    if s.b2 is not None:
        y = y + _float(s.b2)
    if r is not None:
        y = y + r
    y = y.to(s.x.dtype)
    if not s.case["train"]:
        return y
    gy = _float(s.gy)
    gh = gy @ w2.t()
    gz = torch.cat([gh * up * slope, gh * a], dim=1)
    dt = s.x.dtype
    out = [y, (gz @ w1.t()).to(dt), (x.t() @ gz).to(dt), (h.t() @ gy).to(dt)]
    if s.b is not None:
        out += [gz.sum(dim=0).to(dt), gy.sum(dim=0).to(dt)]
    if r is not None:
        out.append(s.gy)
    return out


def run(s):
    c = s.case
    if not own:
        with torch.no_grad():
            return {"norm": _plain_norm, "linear": _plain_linear, "gated": _plain_gated}[c["kind"]](s)
    k = _kernels()
    if c["kind"] == "norm":
        y = k.layer_norm(s.x, s.w, s.b, eps=1e-5)
    elif c["kind"] == "linear":
        y = k.fused_linear(s.x, s.w, s.b, activation=None if c["act"] == "none" else c["act"],
                           residual=s.r)
    else:
        y = k.gated_mlp(s.x, s.w, s.w2, activation=c["act"], bias1=s.b, bias2=s.b2, residual=s.r)
    if not c["train"]:
        return y
    leaves = [t for t in (s.x, s.w, s.w2, s.b, s.b2, s.r) if t is not None]
    return [y.detach(), *torch.autograd.grad(y, leaves, s.gy)]


def work(case):
    """Inputs read once, outputs written once; the products alone as operations
    (a norm's few per value are counted as eight)."""
    size = 4 if case["dtype"] == "f32" else 2
    rows, d, train = case["rows"], case["d"], case["train"]
    if case["kind"] == "norm":
        wt = 0 if case["weights"] == "none" else 4 if case["weights"] == "f32" else size
        # with gradients: the rows, y and its gradient, the rows' gradient
        return {"bytes": rows * d * size * (4 if train else 2) + d * wt * (4 if train else 2),
                "flops": rows * d * (20.0 if train else 8.0)}
    if case["kind"] == "linear":
        n, weights, wide = case["out"], d * case["out"], case["out"]
    else:
        n, weights, wide = d, 3 * d * case["width"], 2 * case["width"] + d
    values = rows * (d + n) + weights
    values += rows * n if case["residual"] else 0
    values += wide if case["bias"] else 0
    if train:  # the output's gradient, and those of every input (the residual's is the output's)
        values += rows * n + rows * d + weights
        values += wide if case["bias"] else 0
    return {"bytes": values * size, "flops": 2.0 * rows * weights * (3 if train else 1)}


def exact(case, seed):
    """The definition in 64 bits, its gradients by autograd."""
    s = prepare(case, seed)
    f = torch.nn.functional

    def wide(t):
        return None if t is None else t.detach().double().requires_grad_(case["train"])

    x, w, b, w2, b2, r = (wide(t) for t in (s.x, s.w, s.b, s.w2, s.b2, s.r))
    acts = {"none": lambda z: z, "relu": torch.relu, "relu_squared": lambda z: torch.relu(z) ** 2,
            "silu": f.silu, "gelu": f.gelu, "gelu_tanh": lambda z: f.gelu(z, approximate="tanh")}
    if case["kind"] == "norm":
        y = f.layer_norm(x, (case["d"],), w, b, 1e-5)
    elif case["kind"] == "linear":
        z = x.matmul(w)
        y = acts[case["act"]](z if b is None else z + b)
    else:
        width = case["width"]
        z = x.matmul(w)
        z = z if b is None else z + b
        y = (acts[GATES[case["act"]]](z[:, :width]) * z[:, width:]).matmul(w2)
        y = y if b2 is None else y + b2
    y = y if r is None else y + r
    if not case["train"]:
        return y
    given = [t for t in (x, w, w2, b, b2, r) if t is not None]
    return [y.detach(), *torch.autograd.grad(y, given, s.gy.double())]

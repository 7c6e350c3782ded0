"""Dense operators beside the expert layer, forward and backward, in bf16 and fp32
(csrc/norm.hip, csrc/dense.hip). The reference has no counterpart: its layer is the
mixture alone (triton_moe/moe.py:42-146).

    y = layer_norm(x, weight, bias)                            # in front of a layer
    y = fused_linear(x, w, bias, "gelu", residual=r)           # act(x w + bias) + r
    y = gated_mlp(x, w1, w2, "swiglu", residual=x)             # a dense block, or an
                                                               # expert of every token

x is [..., features]. Weights are multiplied from the right, w [in, out], in either
order: rows contiguous, or the transposed view of a matrix stored [out, in]
(linear.weight.t()); gradients come in the same order. Calls run on the current
stream of x's device without a host sync, allocate from torch's allocator, record
gradients where autograd does, and can be captured into a graph.
"""

from __future__ import annotations

import functools

import torch

from .. import _lib
from .few_tokens import _on, _untraced

_TYPES = {torch.bfloat16: _lib.DENSE_BF16, torch.float32: _lib.DENSE_F32}
# gated_mlp's activations: that of the gate
_GATES = {"swiglu": "silu", "geglu": "gelu", "geglu_tanh": "gelu_tanh", "reglu": "relu"}
_ACT = _lib.DENSE_ACT


@functools.lru_cache(maxsize=None)
def layer_norm_max() -> int:
    """The longest row layer_norm takes."""
    return int(_lib.lib().vmoe_layer_norm_max())


def _type_of(x, what="x") -> int:
    _lib.require_gpu(x, what)
    code = _TYPES.get(x.dtype)
    if code is None:
        raise NotImplementedError(f"{what} must be bfloat16 or float32 (got {x.dtype})")
    return code


def _rows(t: torch.Tensor, cols: int, mult: int) -> torch.Tensor:
    """t as rows of `cols` values that the kernels read in place where they can:
    [rows, cols] with contiguous 16-byte aligned rows; a copy where not."""
    if t.dim() != 2:
        t = t.reshape(-1, cols)
    if (t.stride(1) != 1 or t.stride(0) % mult or t.data_ptr() % 16 or
            t.stride(0) < cols or t.stride(0) > _MAX_LD):
        t = t.contiguous()
        if t.data_ptr() % 16 or t.stride(0) < cols:  # (a view at an odd place; one row)
            t = t.clone(memory_format=torch.contiguous_format)
    return t


_MAX_LD = 1 << 20


def _weight(w: torch.Tensor, what: str, x: torch.Tensor, mult: int) -> tuple:
    """(weight [in, out] as the kernels read it, leading dimension, transposed)."""
    if w.dim() != 2:
        raise ValueError(f"{what} must have two dimensions (got {w.dim()})")
    if w.dtype != x.dtype:
        raise ValueError(f"{what} must have x's type, {x.dtype} (got {w.dtype})")
    if w.device != x.device:
        raise ValueError(f"{what} must be on x's device, {x.device} (got {w.device})")
    a, b = w.stride()
    if w.data_ptr() % 16 == 0:
        if b == 1 and a >= w.shape[1] and a % mult == 0:
            return w, a, 0
        if a == 1 and b >= w.shape[0] and b % mult == 0:
            return w, b, 1
    # neither order lies as the kernels read it: a copy in the nearer one
    if a == 1 and b != 1:
        c = w.t().clone(memory_format=torch.contiguous_format).t()
        return c, c.stride(1), 1
    c = w.clone(memory_format=torch.contiguous_format)
    return c, c.stride(0), 0


def _vector(v, what: str, n: int, x: torch.Tensor):
    """A bias or norm weight as the kernels read it: [n], bf16 or fp32, contiguous."""
    if v is None:
        return None
    if v.shape != (n,):
        raise ValueError(f"{what} must have shape ({n},) (got {tuple(v.shape)})")
    if v.dtype not in _TYPES:
        raise NotImplementedError(f"{what} must be bfloat16 or float32 (got {v.dtype})")
    if v.device != x.device:
        raise ValueError(f"{what} must be on x's device, {x.device} (got {v.device})")
    return v if v.stride(0) == 1 or n == 1 else v.contiguous()


def _residual(r, shape, x: torch.Tensor):
    if r is None:
        return
    if r.shape != shape:
        raise ValueError(f"residual must have the output's shape {tuple(shape)} "
                         f"(got {tuple(r.shape)})")
    if r.dtype != x.dtype:
        raise ValueError(f"residual must have x's type, {x.dtype} (got {r.dtype})")
    if r.device != x.device:
        raise ValueError(f"residual must be on x's device, {x.device} (got {r.device})")


def _features(x, n: int, what: str, mult: int):
    if n == 0:
        raise ValueError(f"{what} must not be empty")
    if n % mult:
        raise NotImplementedError(f"{what} must be a multiple of {mult} for {x.dtype} "
                                  f"(got {n})")


def _f32(v) -> int:
    return int(v is not None and v.dtype == torch.float32)


def _ptr(v):
    return None if v is None else v.data_ptr()


def _like_weight(shape, transposed: int, w) -> torch.Tensor:
    """An uninitialised gradient of a weight [in, out] in the weight's order."""
    if transposed:
        return torch.empty((shape[1], shape[0]), dtype=w.dtype, device=w.device).t()
    return torch.empty(shape, dtype=w.dtype, device=w.device)


def _ld(g, transposed: int) -> int:
    return g.stride(1) if transposed else g.stride(0)


def _workspace(n: int, device):
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def _recorded(*tensors) -> bool:
    """Whether autograd records a call of these."""
    if not torch.is_grad_enabled():
        return False
    for t in tensors:
        if t is not None and t.requires_grad:
            return True
    return False


# ---------------------------------------------------------------------------
# layer norm


def _norm_rows(x, d: int):
    """x as [rows, d] with contiguous rows at any distance."""
    if x.dim() != 2:
        x = x.reshape(-1, d)
    s = x.stride(0)
    if (x.stride(1) != 1 and d > 1) or (x.shape[0] > 1 and s < d and s != 0):
        x = x.contiguous()
    return x


def _norm_fwd(x, w, b, eps, stats):
    d = x.shape[-1]
    x2 = _norm_rows(x, d)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    rows = x2.shape[0]
    _lib.call("vmoe_layer_norm", _TYPES[x.dtype], x2.data_ptr(), x2.stride(0) if rows > 1 else d,
              rows, d, _ptr(w), _f32(w), _ptr(b), _f32(b), eps, y.data_ptr(), d, _ptr(stats),
              _lib.stream(x.device))
    return y


class LayerNormOp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, eps):
        with _on(x.device):
            rows = x.numel() // x.shape[-1]
            stats = torch.empty((rows, 2), dtype=torch.float32, device=x.device)
            y = _norm_fwd(x, w, b, eps, stats)
        ctx.save_for_backward(x, w, b, stats)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy):
        x, w, b, stats = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        with _on(x.device):
            return (*_norm_bwd(gy, x, w, b, stats, need_x, need_w, need_b), None)


def _norm_bwd(gy, x, w, b, stats, need_x, need_w, need_b):
    d, rows = x.shape[-1], stats.shape[0]
    gx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_x else None
    gw = torch.empty_like(w, memory_format=torch.contiguous_format) if need_w else None
    gb = torch.empty_like(b, memory_format=torch.contiguous_format) if need_b else None
    if rows == 0:
        for g in (gw, gb):
            if g is not None:
                g.zero_()
        return gx, gw, gb
    x2, g2 = _norm_rows(x, d), _norm_rows(gy, d)
    n = int(_lib.lib().vmoe_layer_norm_workspace_bytes(rows, d)) if need_w or need_b else 0
    ws = _workspace(n, x.device)
    _lib.call("vmoe_layer_norm_backward", _TYPES[x.dtype], g2.data_ptr(),
              g2.stride(0) if rows > 1 else d, x2.data_ptr(), x2.stride(0) if rows > 1 else d,
              rows, d, _ptr(w), _f32(w), stats.data_ptr(), _ptr(gx), d, _ptr(gw), _f32(gw),
              _ptr(gb), _f32(gb), _ptr(ws), n, _lib.stream(x.device))
    return gx, gw, gb


@_untraced
def layer_norm(x, weight=None, bias=None, eps: float = 1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension of x
    [..., d], 1 to layer_norm_max() values, of any size and row distance. x is bf16 or
    fp32 and so is the output; weight and bias [d] may be of either type each.
    Statistics and sums are fp32."""
    _type_of(x)
    if x.dim() == 0:
        raise ValueError("x must have at least one dimension")
    d = x.shape[-1]
    if d == 0:
        raise ValueError("the last dimension of x must not be empty")
    if d > layer_norm_max():
        raise NotImplementedError(f"rows of at most {layer_norm_max()} values (got {d})")
    w, b = _vector(weight, "weight", d, x), _vector(bias, "bias", d, x)
    if _recorded(x, w, b):
        return LayerNormOp.apply(x, w, b, eps)
    with _on(x.device):
        return _norm_fwd(x, w, b, eps, None)


# ---------------------------------------------------------------------------
# linear layer with a fused epilogue


def _linear_fwd(x2, wt, ldw, tr, b, act, r, out, keep):
    """(y [rows, out], z or None): keep: whether the backward pass needs z."""
    rows, d = x2.shape
    code = _TYPES[x2.dtype]
    dev = x2.device
    y = torch.empty((rows, out), dtype=x2.dtype, device=dev)
    z = torch.empty((rows, out), dtype=torch.float32, device=dev) if keep else None
    r2 = None if r is None else _rows(r, out, 16 // x2.element_size())
    n = _linear_bytes(code, rows, d, out, act, 0)
    ws = _workspace(n, dev)
    _lib.call("vmoe_linear_forward", code, x2.data_ptr(), x2.stride(0), rows, d, out,
              wt.data_ptr(), ldw, tr, _ptr(b), _f32(b), act, _ptr(r2),
              0 if r2 is None else r2.stride(0), y.data_ptr(), out, _ptr(z), _ptr(ws), n,
              _lib.stream(dev))
    return y, z


@functools.lru_cache(maxsize=4096)
def _linear_bytes(code, rows, d, out, act, backward) -> int:
    return int(_lib.lib().vmoe_linear_workspace_bytes(code, rows, d, out, act, backward))


class FusedLinearOp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, r, act):
        d, out = w.shape
        mult = 16 // x.element_size()
        with _on(x.device):
            x2 = _rows(x, d, mult)
            wt, ldw, tr = _weight(w, "weight", x, mult)
            y, z = _linear_fwd(x2, wt, ldw, tr, b, act, r, out, act != 0)
        ctx.save_for_backward(x, w, b, z)
        ctx.act = act
        return y.view(*x.shape[:-1], out)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy):
        x, w, b, z = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        gx = gw = gb = None
        if need_x or need_w or need_b:
            with _on(x.device):
                gx, gw, gb = _linear_bwd(gy, x, w, b, z, ctx.act, need_x, need_w, need_b)
        return gx, gw, gb, gy if need_r else None, None


def _linear_bwd(gy, x, w, b, z, act, need_x, need_w, need_b):
    d, out = w.shape
    dev, mult = x.device, 16 // x.element_size()
    wt, ldw, tr = _weight(w, "weight", x, mult)
    gx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
    gw = _like_weight((d, out), tr, w) if need_w else None
    gb = torch.empty(out, dtype=b.dtype, device=dev) if need_b else None
    if x.numel() == 0:
        for g in (gw, gb):
            if g is not None:
                g.zero_()
        return gx, gw, gb
    x2, g2 = _rows(x, d, mult), _rows(gy, out, mult)
    rows, code = x2.shape[0], _TYPES[x.dtype]
    n = _linear_bytes(code, rows, d, out, act, 1)
    ws = _workspace(n, dev)
    _lib.call("vmoe_linear_backward", code, g2.data_ptr(), g2.stride(0), x2.data_ptr(),
              x2.stride(0), rows, d, out, wt.data_ptr(), ldw, tr, act, _ptr(z), _ptr(gx), d,
              _ptr(gw), 0 if gw is None else _ld(gw, tr), _ptr(gb), _f32(gb), _ptr(ws), n,
              _lib.stream(dev))
    return gx, gw, gb


@_untraced
def fused_linear(x, weight, bias=None, activation=None, residual=None):
    """activation(x weight + bias) + residual in one product: x [..., in], weight
    [in, out], bias [out], residual of the output's shape and type. activation: None,
    "relu", "relu_squared", "silu", "gelu" or "gelu_tanh". x and weight are bf16 or fp32
    (the same), bias either; in and out multiples of 8 (fp32: 4). Sums, bias,
    activation and residual are fp32, the output is rounded once. With an activation the
    backward pass keeps x weight + bias in fp32."""
    _type_of(x)
    if activation not in _ACT:
        raise ValueError(f"Unknown activation: {activation} (expected one of "
                         f"{sorted(a for a in _ACT if a)} or None)")
    if x.dim() == 0 or weight.dim() != 2 or x.shape[-1] != weight.shape[0]:
        raise ValueError(f"x [..., in] and weight [in, out] do not fit: {tuple(x.shape)}, "
                         f"{tuple(weight.shape)}")
    d, out = weight.shape
    mult = 16 // x.element_size()
    _features(x, d, "in", mult)
    _features(x, out, "out", mult)
    b = _vector(bias, "bias", out, x)
    _residual(residual, (*x.shape[:-1], out), x)
    act = _ACT[activation]
    if _recorded(x, weight, b, residual):
        _weight(weight, "weight", x, mult)
        return FusedLinearOp.apply(x, weight, b, residual, act)
    with _on(x.device):
        wt, ldw, tr = _weight(weight, "weight", x, mult)
        y, _ = _linear_fwd(_rows(x, d, mult), wt, ldw, tr, b, act, residual, out, False)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], out)


# ---------------------------------------------------------------------------
# gated block


@functools.lru_cache(maxsize=4096)
def _gated_bytes(code, rows, d, width, backward) -> int:
    return int(_lib.lib().vmoe_gated_workspace_bytes(code, rows, d, width, backward))


def _gated_fwd(x2, a1, a2, b1, b2, act, r, keep):
    """(y, h, z or None)."""
    (w1, ld1, t1), (w2, ld2, t2) = a1, a2
    rows, d = x2.shape
    width, dev, code = w2.shape[0], x2.device, _TYPES[x2.dtype]
    y = torch.empty((rows, d), dtype=x2.dtype, device=dev)
    h = torch.empty((rows, width), dtype=x2.dtype, device=dev)
    z = torch.empty((rows, 2 * width), dtype=torch.float32, device=dev) if keep else None
    r2 = None if r is None else _rows(r, d, 16 // x2.element_size())
    n = _gated_bytes(code, rows, d, width, 0)
    ws = _workspace(n, dev)
    _lib.call("vmoe_gated_forward", code, x2.data_ptr(), x2.stride(0), rows, d, width,
              w1.data_ptr(), ld1, t1, _ptr(b1), _f32(b1), act, w2.data_ptr(), ld2, t2, _ptr(b2),
              _f32(b2), _ptr(r2), 0 if r2 is None else r2.stride(0), h.data_ptr(), _ptr(z),
              y.data_ptr(), d, _ptr(ws), n, _lib.stream(dev))
    return y, h, z


class GatedMLPOp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w1, w2, b1, b2, r, act):
        mult = 16 // x.element_size()
        with _on(x.device):
            y, h, z = _gated_fwd(_rows(x, x.shape[-1], mult), _weight(w1, "w1", x, mult),
                                 _weight(w2, "w2", x, mult), b1, b2, act, r, True)
        ctx.save_for_backward(x, w1, w2, b1, b2, h, z)
        ctx.act = act
        return y.view(x.shape)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy):
        need = ctx.needs_input_grad
        grads = (None,) * 5
        if any(need[:5]):
            x = ctx.saved_tensors[0]
            with _on(x.device):
                grads = _gated_bwd(gy, *ctx.saved_tensors, ctx.act, need)
        return (*grads, gy if need[5] else None, None)


def _gated_bwd(gy, x, w1, w2, b1, b2, h, z, act, need):
    width, d = w2.shape
    dev, mult, code = x.device, 16 // x.element_size(), _TYPES[x.dtype]
    (a1, ld1, t1), (a2, ld2, t2) = _weight(w1, "w1", x, mult), _weight(w2, "w2", x, mult)
    gx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need[0] else None
    gw1 = _like_weight((d, 2 * width), t1, w1) if need[1] else None
    gw2 = _like_weight((width, d), t2, w2) if need[2] else None
    gb1 = torch.empty(2 * width, dtype=b1.dtype, device=dev) if need[3] else None
    gb2 = torch.empty(d, dtype=b2.dtype, device=dev) if need[4] else None
    if x.numel() == 0:
        for g in (gw1, gw2, gb1, gb2):
            if g is not None:
                g.zero_()
        return gx, gw1, gw2, gb1, gb2
    x2, g2 = _rows(x, d, mult), _rows(gy, d, mult)
    rows = x2.shape[0]
    n = _gated_bytes(code, rows, d, width, 1)
    ws = _workspace(n, dev)
    _lib.call("vmoe_gated_backward", code, g2.data_ptr(), g2.stride(0), x2.data_ptr(),
              x2.stride(0), rows, d, width, a1.data_ptr(), ld1, t1, a2.data_ptr(), ld2, t2, act,
              h.data_ptr(), z.data_ptr(), _ptr(gx), d, _ptr(gw1),
              0 if gw1 is None else _ld(gw1, t1), _ptr(gb1), _f32(gb1), _ptr(gw2),
              0 if gw2 is None else _ld(gw2, t2), _ptr(gb2), _f32(gb2), _ptr(ws), n,
              _lib.stream(dev))
    return gx, gw1, gw2, gb1, gb2


@_untraced
def gated_mlp(x, w1, w2, activation="swiglu", bias1=None, bias2=None, residual=None):
    """A gated feed-forward block: with [g | u] = x w1 + bias1 and h = act(g) * u,
    h w2 + bias2 + residual. x [..., d], w1 [d, 2 width] (gates, then ups), w2 [width, d],
    bias1 [2 width], bias2 [d], residual of x's shape and type. activation: "swiglu" (silu
    on the gate), "geglu", "geglu_tanh" or "reglu". Both projections, the activation and
    the product are one launch, the second product with bias and residual another. x and
    the weights are bf16 or fp32 (the same), biases either; d and width multiples of 8
    (fp32: 4). h is rounded to x's type, as an operand of the second product; the
    backward pass keeps g and u in fp32."""
    _type_of(x)
    if activation not in _GATES:
        raise ValueError(f"Unknown activation: {activation} (expected one of {sorted(_GATES)})")
    if (x.dim() == 0 or w1.dim() != 2 or w2.dim() != 2 or x.shape[-1] != w1.shape[0] or
            w2.shape[1] != w1.shape[0] or w1.shape[1] != 2 * w2.shape[0]):
        raise ValueError(f"x [..., d], w1 [d, 2 width] and w2 [width, d] do not fit: "
                         f"{tuple(x.shape)}, {tuple(w1.shape)}, {tuple(w2.shape)}")
    width, d = w2.shape
    mult = 16 // x.element_size()
    _features(x, d, "d", mult)
    _features(x, width, "width", mult)
    b1, b2 = _vector(bias1, "bias1", 2 * width, x), _vector(bias2, "bias2", d, x)
    _residual(residual, x.shape, x)
    act = _ACT[_GATES[activation]]
    if _recorded(x, w1, w2, b1, b2, residual):
        for w, n in ((w1, "w1"), (w2, "w2")):
            _weight(w, n, x, mult)
        return GatedMLPOp.apply(x, w1, w2, b1, b2, residual, act)
    with _on(x.device):
        y, _, _ = _gated_fwd(_rows(x, d, mult), _weight(w1, "w1", x, mult),
                             _weight(w2, "w2", x, mult), b1, b2, act, residual, False)
    return y if x.dim() == 2 else y.view(x.shape)

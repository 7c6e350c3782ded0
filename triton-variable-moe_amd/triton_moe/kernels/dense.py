"""Dense operators beside the expert layer, forward and backward, in bf16 and fp32
(csrc/norm.hip, csrc/dense.hip; called through csrc/dense_torch.cpp). The reference has
no counterpart: its layer is the mixture alone (triton_moe/moe.py:42-146).

    y = layer_norm(x, weight, bias)                            # in front of a layer
    y = fused_linear(x, w, bias, "gelu", residual=r)           # act(x w + bias) + r
    y = gated_mlp(x, w1, w2, "swiglu", residual=x)             # a dense block, or an
                                                               # expert of every token

x is [..., features]. Weights are multiplied from the right, w [in, out], in either
order: rows contiguous, or the transposed view of a matrix stored [out, in]
(linear.weight.t()); gradients come in the same order. Tensors that the kernels cannot
read in place (rows not contiguous, or not aligned to 16 bytes) are copied. Calls run
on the current stream of x's device without a host sync, allocate from torch's
allocator, record gradients where autograd does, and can be captured into a graph. A
recorded call saves what the gradients that can be asked for read (no pre-activations
for a residual's or w2's, no x where the weight takes none; layer_norm always x).
Gradients cannot be differentiated again, and there are no forward-mode derivatives.
"""

from __future__ import annotations

import functools

from .. import _lib
from .few_tokens import _untraced

# gated_mlp's activations: that of the gate
_GATES = {"swiglu": "silu", "geglu": "gelu", "geglu_tanh": "gelu_tanh", "reglu": "relu"}
_ACT = _lib.DENSE_ACT
_GATE_ACT = {name: _ACT[gate] for name, gate in _GATES.items()}


@functools.lru_cache(maxsize=None)
def layer_norm_max() -> int:
    """The longest row layer_norm takes."""
    return int(_lib.lib().vmoe_layer_norm_max())


@_untraced
def layer_norm(x, weight=None, bias=None, eps: float = 1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension of x
    [..., d], 1 to layer_norm_max() values, of any size and row distance. x is bf16 or
    fp32 and so is the output; weight and bias [d] may be of either type each.
    Statistics and sums are fp32."""
    return _lib.dense().layer_norm(x, weight, bias, eps)


@_untraced
def fused_linear(x, weight, bias=None, activation=None, residual=None):
    """activation(x weight + bias) + residual in one product: x [..., in], weight
    [in, out], bias [out], residual of the output's shape and type. activation: None,
    "relu", "relu_squared", "silu", "gelu" or "gelu_tanh". x and weight are bf16 or fp32
    (the same), bias either; in and out multiples of 8 (fp32: 4). Sums, bias,
    activation and residual are fp32, the output is rounded once. With an activation
    x weight + bias is kept in fp32 for the backward pass; with relu and no residual the
    output is kept instead (it must not be changed in place). The gradient through the
    activation is rounded to x's type, as an operand of the gradients' products."""
    act = _ACT.get(activation)
    if act is None:
        raise ValueError(f"Unknown activation: {activation} (expected one of "
                         f"{sorted(a for a in _ACT if a)} or None)")
    return _lib.dense().fused_linear(x, weight, bias, residual, act)


@_untraced
def gated_mlp(x, w1, w2, activation="swiglu", bias1=None, bias2=None, residual=None):
    """A gated feed-forward block: with [g | u] = x w1 + bias1 and h = act(g) * u,
    h w2 + bias2 + residual. x [..., d], w1 [d, 2 width] (gates, then ups), w2 [width, d],
    bias1 [2 width], bias2 [d], residual of x's shape and type. activation: "swiglu" (silu
    on the gate), "geglu", "geglu_tanh" or "reglu". Both projections, the activation and
    the product are one kernel, the second product with bias and residual another. x and
    the weights are bf16 or fp32 (the same), biases either; d and width multiples of 8
    (fp32: 4). h is rounded to x's type, as an operand of the second product, and so are
    the gradients of g and u; the backward pass keeps g and u in fp32."""
    act = _GATE_ACT.get(activation)
    if act is None:
        raise ValueError(f"Unknown activation: {activation} (expected one of {sorted(_GATES)})")
    return _lib.dense().gated_mlp(x, w1, w2, bias1, bias2, residual, act)

"""Refusals of the dense operators, through torch and at the C entry points, on the
host: no call here reaches a launch."""

from __future__ import annotations

import pytest
import torch

from triton_moe import _lib
from triton_moe import kernels as K

P = 0x1000  # an aligned address that nothing here reads
OK, BAD, NOT, WS = _lib.OK, _lib.ERR_INVALID_ARG, _lib.ERR_UNSUPPORTED, _lib.ERR_WORKSPACE
HUGE = 1 << 60


def t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


BF16, F16, F64 = torch.bfloat16, torch.float16, torch.float64


@pytest.mark.parametrize("call,error,text", [
    (lambda: K.layer_norm(t(3, 8, dtype=F16)), NotImplementedError, "bfloat16 or float32"),
    (lambda: K.layer_norm(t(3, 8, dtype=torch.int32)), NotImplementedError, "bfloat16 or float32"),
    (lambda: K.layer_norm(t()), ValueError, "at least one dimension"),
    (lambda: K.layer_norm(t(3, 0)), ValueError, "must not be empty"),
    (lambda: K.layer_norm(t(1, K.layer_norm_max() + 1)), NotImplementedError, "at most"),
    (lambda: K.layer_norm(t(3, 8), t(7)), ValueError, r"weight must have shape \(8,\)"),
    (lambda: K.layer_norm(t(3, 8), t(1, 8)), ValueError, "weight must have shape"),
    (lambda: K.layer_norm(t(3, 8), None, t(9)), ValueError, "bias must have shape"),
    (lambda: K.layer_norm(t(3, 8), t(8, dtype=F64)), NotImplementedError, "weight must be bfloat16"),
    (lambda: K.layer_norm([1.0]), TypeError, "x must be a tensor"),
    (lambda: K.layer_norm(t(3, 8), 1.0), TypeError, "weight must be a tensor"),
    (lambda: K.layer_norm(t(3, 8), eps="1"), TypeError, ""),
    (lambda: K.layer_norm(t(3, 8).to_sparse()), NotImplementedError, "strided"),
    (lambda: K.layer_norm(t(3, 8)), AssertionError, "x must be on CUDA"),
    (lambda: K.fused_linear(t(3, 8, dtype=F16), t(8, 8, dtype=F16)), NotImplementedError, "bfloat16"),
    (lambda: K.fused_linear(t(3, 8), t(8, 8), activation="tanh"), ValueError, "Unknown activation"),
    (lambda: K.fused_linear(t(3, 8), t(8, 8), activation="swiglu"), ValueError, "Unknown activation"),
    (lambda: K.fused_linear(t(3, 8), t(16, 8)), ValueError, "do not fit"),
    (lambda: K.fused_linear(t(3, 8), t(8)), ValueError, "do not fit"),
    (lambda: K.fused_linear(t(), t(8, 8)), ValueError, "do not fit"),
    (lambda: K.fused_linear(t(3, 0), t(0, 8)), ValueError, "in must not be empty"),
    (lambda: K.fused_linear(t(3, 8), t(8, 0)), ValueError, "out must not be empty"),
    (lambda: K.fused_linear(t(3, 6), t(6, 8)), NotImplementedError, "in must be a multiple of 4"),
    (lambda: K.fused_linear(t(3, 12, dtype=BF16), t(12, 8, dtype=BF16)), NotImplementedError,
     "in must be a multiple of 8"),
    (lambda: K.fused_linear(t(3, 8, dtype=BF16), t(8, 12, dtype=BF16)), NotImplementedError,
     "out must be a multiple of 8"),
    (lambda: K.fused_linear(t(3, 8, dtype=BF16), t(8, 8)), ValueError, "weight must have x's type"),
    (lambda: K.fused_linear(t(3, 8), t(8, 12), t(8)), ValueError, "bias must have shape"),
    (lambda: K.fused_linear(t(3, 8), t(8, 12), t(12, dtype=F16)), NotImplementedError, "bias must be"),
    (lambda: K.fused_linear(t(3, 8), t(8, 12), residual=t(3, 8)), ValueError,
     "residual must have the output's shape"),
    (lambda: K.fused_linear(t(3, 8), t(8, 12), residual=t(12)), ValueError, "residual must have"),
    (lambda: K.fused_linear(t(3, 8), t(8, 12), residual=t(3, 12, dtype=BF16)), ValueError,
     "residual must have x's type"),
    (lambda: K.fused_linear(t(3, 8), t(8, 12)), AssertionError, "x must be on CUDA"),
    (lambda: K.gated_mlp(t(3, 8), t(8, 32), t(16, 8), "silu"), ValueError, "Unknown activation"),
    (lambda: K.gated_mlp(t(3, 8), t(8, 32), t(16, 8), None), ValueError, "Unknown activation"),
    (lambda: K.gated_mlp(t(3, 8), t(8, 16), t(16, 8)), ValueError, "do not fit"),
    (lambda: K.gated_mlp(t(3, 8), t(8, 32), t(16, 12)), ValueError, "do not fit"),
    (lambda: K.gated_mlp(t(3, 8), t(8, 28, dtype=F64), t(14, 8)), NotImplementedError,
     "width must be a multiple of 4"),
    (lambda: K.gated_mlp(t(3, 8), t(8, 0), t(0, 8)), ValueError, "width must not be empty"),
    (lambda: K.gated_mlp(t(3, 8), t(8, 32), t(16, 8, dtype=BF16)), ValueError, "w2 must have x's type"),
    (lambda: K.gated_mlp(t(3, 8), t(8, 32), t(16, 8), bias1=t(16)), ValueError, "bias1 must have"),
    (lambda: K.gated_mlp(t(3, 8), t(8, 32), t(16, 8), bias2=t(16)), ValueError, "bias2 must have"),
    (lambda: K.gated_mlp(t(3, 8), t(8, 32), t(16, 8), residual=t(4, 8)), ValueError, "residual must"),
    (lambda: K.gated_mlp(t(3, 8), t(8, 32), t(16, 8)), AssertionError, "x must be on CUDA"),
])
def test_calls_are_checked(call, error, text):
    with pytest.raises(error, match=text):
        call()


def norm(type=0, x=P, ldx=64, rows=2, d=64, w=P, b=P, y=P, ldy=64, stats=None):
    return _lib.lib().vmoe_layer_norm(type, x, ldx, rows, d, w, 0, b, 0, 1e-5, y, ldy, stats, None)


def norm_bwd(type=0, gy=P, ldgy=64, x=P, ldx=64, rows=2, d=64, stats=P, gx=P, ldgx=64, gw=P, gb=P,
             ws=P, n=HUGE):
    if n == "short":
        n = _lib.lib().vmoe_layer_norm_workspace_bytes(rows, d) - 1
    return _lib.lib().vmoe_layer_norm_backward(type, gy, ldgy, x, ldx, rows, d, P, 0, stats, gx, ldgx,
                                               gw, 0, gb, 0, ws, n, None)


@pytest.mark.parametrize("change,status", [
    (dict(rows=0), OK), (dict(type=2), BAD), (dict(type=-1), BAD), (dict(rows=-1), BAD),
    (dict(d=0), BAD), (dict(d=-64), BAD), (dict(d=1 << 20, ldx=1 << 20), NOT), (dict(x=None), BAD),
    (dict(ldx=-64), BAD), (dict(ldx=63), BAD), (dict(ldy=63), BAD), (dict(stats=P + 4), NOT),
    (dict(y=None), BAD),
])
def test_layer_norm_entry(change, status):
    assert norm(**change) == status


@pytest.mark.parametrize("change,status", [
    (dict(rows=0), OK), (dict(gx=None, gw=None, gb=None), OK), (dict(type=2), BAD), (dict(d=0), BAD),
    (dict(rows=-2), BAD), (dict(x=None), BAD), (dict(gy=None), BAD), (dict(stats=None), BAD),
    (dict(stats=P + 4), NOT), (dict(ldgy=63), BAD), (dict(ldgy=-1), BAD), (dict(ldx=63), BAD),
    (dict(ldgx=63), BAD), (dict(ws=None), BAD), (dict(n=0), WS), (dict(ws=P + 8), NOT),
    (dict(n="short"), WS),
])
def test_layer_norm_backward_entry(change, status):
    assert norm_bwd(**change) == status


def linear(type=0, x=P, ldx=64, rows=2, i=64, o=64, w=P, ldw=64, tr=0, act=0, r=None, ldr=64, y=P,
           ldy=64, z=None, ws=P, n=HUGE, words=None):
    return _lib.lib().vmoe_linear_forward(type, x, ldx, rows, i, o, w, ldw, tr, None, 0, act, r, ldr, y,
                                          ldy, z, ws, n, words, None)


SIZES = [(dict(type=2), BAD), (dict(act=6), BAD), (dict(act=-1), BAD), (dict(rows=-1), BAD),
         (dict(rows=(1 << 22) + 1), NOT)]


@pytest.mark.parametrize("change,status", SIZES + [
    (dict(rows=0), OK), (dict(i=0), BAD), (dict(o=0), BAD), (dict(i=60), NOT), (dict(o=60), NOT),
    (dict(type=1, i=62), NOT), (dict(x=None), BAD), (dict(ldx=56), BAD), (dict(ldx=68), NOT),
    (dict(x=P + 8), NOT), (dict(ldx=(1 << 20) + 8), NOT), (dict(w=None), BAD), (dict(w=P + 2), NOT),
    (dict(ldw=56), BAD), (dict(ldw=60), BAD), (dict(o=128, ldw=64, ldy=128), BAD),
    (dict(i=128, ldx=128, tr=1, ldw=64), BAD), (dict(ldw=(1 << 20) + 8), NOT), (dict(y=None), BAD),
    (dict(ldy=56), BAD), (dict(y=P + 4), NOT), (dict(r=P, ldr=56), BAD), (dict(r=P + 2), NOT),
    (dict(z=P + 8), NOT), (dict(words=P + 2), NOT),
])
def test_linear_entry(change, status):
    assert linear(**change) == status


def linear_bwd(type=0, gy=P, ldgy=64, x=P, ldx=64, rows=2, i=64, o=64, w=P, ldw=64, tr=0, act=0,
               z=None, y=None, ldy=64, gx=P, ldgx=64, gw=P, ldgw=64, gb=P, ws=P, n=HUGE):
    if n == "short":
        n = _lib.lib().vmoe_linear_workspace_bytes(type, rows, i, o, act, 1) - 1
    return _lib.lib().vmoe_linear_backward(type, gy, ldgy, x, ldx, rows, i, o, w, ldw, tr, act, z, y,
                                           ldy, gx, ldgx, gw, ldgw, gb, 0, ws, n, None)


@pytest.mark.parametrize("change,status", SIZES + [
    (dict(rows=0), OK), (dict(gy=None), BAD), (dict(ldgy=56), BAD), (dict(x=None), BAD),
    (dict(w=None), BAD), (dict(ldgx=56), BAD), (dict(gx=P + 8), NOT), (dict(gw=P + 8), NOT),
    (dict(ldgw=56), BAD), (dict(act=1), BAD), (dict(act=1, z=P + 4), NOT),
    (dict(act=3, y=P), BAD), (dict(act=2, y=P), BAD), (dict(act=1, y=P, ldy=56), BAD),
    (dict(act=1, y=P + 8), NOT), (dict(n=0), WS),
    (dict(ws=None), BAD), (dict(ws=P + 8), NOT),
    (dict(n="short"), WS),
])
def test_linear_backward_entry(change, status):
    assert linear_bwd(**change) == status


def gated(type=0, x=P, ldx=64, rows=2, d=64, width=32, w1=P, ldw1=64, t1=0, act=3, w2=P, ldw2=64, t2=0,
          r=None, ldr=64, h=P, z=None, y=P, ldy=64, ws=P, n=HUGE, words=None):
    return _lib.lib().vmoe_gated_forward(type, x, ldx, rows, d, width, w1, ldw1, t1, None, 0, act, w2,
                                         ldw2, t2, None, 0, r, ldr, h, z, y, ldy, ws, n, words, None)


@pytest.mark.parametrize("change,status", SIZES + [
    (dict(rows=0), OK), (dict(d=0), BAD), (dict(width=0), BAD), (dict(width=28, ldw1=56), NOT),
    (dict(x=None), BAD), (dict(w1=None), BAD), (dict(ldw1=56), BAD), (dict(w2=None), BAD),
    (dict(ldw2=56), BAD), (dict(t2=1, ldw2=24), BAD), (dict(h=None), BAD), (dict(h=P + 8), NOT),
    (dict(y=None), BAD), (dict(z=P + 8), NOT), (dict(r=P + 8), NOT), (dict(ldr=56, r=P), BAD),
    (dict(words=P + 1), NOT),
    # the ups of a weight stored [2 width, hidden] lie 2 GiB behind the gates
    (dict(t1=1, ldw1=1 << 20, width=1024), NOT),
])
def test_gated_entry(change, status):
    assert gated(**change) == status


def gated_bwd(type=0, gy=P, ldgy=64, x=P, rows=2, d=64, width=32, ldw1=64, t1=0, act=3, h=P, z=P, gx=P,
              gw1=P, ldgw1=64, gb1=P, gw2=P, ldgw2=64, gb2=P, ws=P, n=HUGE):
    if n == "short":
        n = _lib.lib().vmoe_gated_workspace_bytes(type, rows, d, width, 1) - 1
    return _lib.lib().vmoe_gated_backward(type, gy, ldgy, x, 64, rows, d, width, P, ldw1, t1, P, 64, 0,
                                          act, h, z, gx, 64, gw1, ldgw1, gb1, 0, gw2, ldgw2, gb2, 0, ws,
                                          n, None)


@pytest.mark.parametrize("change,status", SIZES + [
    (dict(rows=0), OK), (dict(gy=None), BAD), (dict(ldgy=56), BAD), (dict(z=None), BAD),
    (dict(z=P + 8), NOT), (dict(h=None), BAD), (dict(x=None), BAD), (dict(gx=P + 8), NOT),
    (dict(gw1=P + 8), NOT), (dict(ldgw1=56), BAD), (dict(gw2=P + 8), NOT), (dict(ldgw2=56), BAD),
    (dict(n=0), WS), (dict(ws=None), BAD), (dict(t1=1, ldw1=1 << 20, width=1024), NOT),
    (dict(n="short"), WS),
])
def test_gated_backward_entry(change, status):
    assert gated_bwd(**change) == status


def test_workspace_queries():
    """No workspace of sizes that are refused; one that grows with what is asked for."""
    lib = _lib.lib()
    assert lib.vmoe_linear_workspace_bytes(0, 2, 60, 64, 0, 1) == 0
    assert lib.vmoe_linear_workspace_bytes(3, 2, 64, 64, 0, 1) == 0
    assert lib.vmoe_gated_workspace_bytes(0, 2, 64, -8, 0) == 0
    assert lib.vmoe_layer_norm_workspace_bytes(2, lib.vmoe_layer_norm_max() + 1) == 0
    a = lib.vmoe_linear_workspace_bytes(0, 256, 512, 512, 0, 1)
    b = lib.vmoe_linear_workspace_bytes(0, 256, 512, 512, 3, 1)
    assert b == a + 256 * 512 * 2  # the gradient through the activation
    # the largest sizes: in 64 bits
    n = lib.vmoe_gated_workspace_bytes(1, 1 << 22, 1 << 16, 1 << 16, 1)
    assert n > (1 << 22) * (1 << 17) * 4

"""The activations of the dense operators, and their slopes, where they are saturated:
arguments of 30 and more, up to the largest numbers, against 64 bits.

Bounds, u = 2^-24. There an activation is z, z^2, 0 or z times a small exponential, its
slope 1, 2 z, 0 or such an exponential: a few operations, 16 u of the value. A sigmoid
below the smallest normal number may be 0: |z| 2^-126. Then the rounding of what is stored
in the rows' type, for a gradient also that of the product's operand.
"""

from __future__ import annotations

import pytest
import torch

from test_gpu_dense import ACTS, GATES
from triton_moe import kernels as K

pytestmark = pytest.mark.gpu

U, TINY = 2.0 ** -24, 2.0 ** -126
SIZES = [30.0, 45.0, 87.0, 89.0, 104.0, 1e3, 1e4, 3e9, 1e13, 1e16, 1.7e19, 1.9e19, 1e20, 1e30, 3e38]


def arguments(dtype):
    v = torch.tensor(SIZES)
    return torch.cat([v, -v]).to(dtype)


def reference(act, z):
    z = z.double().requires_grad_()
    y = ACTS[act](z)
    return y.detach(), torch.autograd.grad(y.sum(), z)[0]


def hold(got, ref, z, roundings, what):
    got, z = got.detach().cpu().double(), z.double()
    big = torch.finfo(what[-1]).max
    over = ref.abs() > big  # past the type's range
    assert torch.equal(got[over], ref[over].sign() * float("inf")), what
    tol = (16 * U + roundings * torch.finfo(what[-1]).eps / 2) * ref.abs() + z.abs() * TINY
    d = (got - ref).abs()
    assert (d <= tol)[~over].all(), (what, z[~over][~(d <= tol)[~over]], got[~over][~(d <= tol)[~over]])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", list(ACTS))
def test_fused_linear(act, dtype, device):
    z = arguments(dtype)
    x = torch.zeros(z.numel(), 8, dtype=dtype)
    x[:, 0] = z
    x = x.cuda().requires_grad_()
    w = torch.zeros(8, 8, dtype=dtype)
    w[0, 0] = 1.0
    gy = torch.zeros(z.numel(), 8, dtype=dtype)
    gy[:, 0] = 1.0
    zero = torch.zeros(z.numel(), 8, dtype=dtype).cuda()
    ref, slope = reference(act, z)
    for r in (None, zero):  # (relu's slope comes from the output, or from the sums)
        y = K.fused_linear(x, w.cuda(), None, act, r)
        gx, = torch.autograd.grad(y, x, gy.cuda())
        hold(y[:, 0], ref, z, 1, ("y", dtype))
        hold(gx[:, 0], slope, z, 2, ("x.grad", dtype))
        # (2 z of 3e38 is past every range: infinity, whose products with the other
        # weights' zeros are NaN)
        fits = slope.abs().cuda() <= torch.finfo(dtype).max
        assert not y[:, 1:].any() and not gx[fits, 1:].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", sorted(GATES))
def test_gated_mlp(act, dtype, device):
    z = arguments(dtype)
    for rows in (z, z.repeat(30)):  # few rows, and tiles
        x = torch.zeros(rows.numel(), 8, dtype=dtype)
        x[:, 0] = rows
        x = x.cuda().requires_grad_()
        w1, w2 = torch.zeros(8, 16, dtype=dtype), torch.zeros(8, 8, dtype=dtype)
        w1[0, 0] = w2[0, 0] = 1.0
        b1 = torch.zeros(16)
        b1[8] = 1.0  # the up half
        gy = torch.zeros(rows.numel(), 8, dtype=dtype)
        gy[:, 0] = 1.0
        ref, slope = reference(GATES[act], rows)
        y = K.gated_mlp(x, w1.cuda(), w2.cuda(), act, b1.cuda())
        gx, = torch.autograd.grad(y, x, gy.cuda())
        hold(y[:, 0], ref, rows, 2, ("y", dtype))
        hold(gx[:, 0], slope, rows, 2, ("x.grad", dtype))

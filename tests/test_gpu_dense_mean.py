"""Layer norm of rows whose spread is small beside their mean, against 64 bits.

Bounds. u = 2^-24; a sum over a row is off by at most K u times the sum of its terms'
sizes (K = 64: 16 additions in a thread, 6 across a wave, 16 across waves, few around).
The first mean m' is off by e0 = K u mean|x|. The values c = x - m' are rounded once, and
their mean, which is what m' is off by, is taken out again: what stays is at most
E = K u (mean|x - m| + e0) and two roundings of a value. The variance is the mean of the
squares of what stays, off by K u of itself and E^2. The mean is kept as one float for the
backward pass, which rounds it: u |m|, divided by the deviation.
"""

from __future__ import annotations

import pytest
import torch

from triton_moe import kernels as K

pytestmark = pytest.mark.gpu

U, KS = 2.0 ** -24, 64
BF16, F32 = torch.bfloat16, torch.float32


def wide(t):
    return t.detach().cpu().double()


def reference(x, w, b, gy, eps):
    x, w, b, gy = (wide(t) for t in (x, w, b, gy))
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    var = (c * c).mean(-1, keepdim=True) + eps
    rstd = var ** -0.5
    xh = c * rstd
    y = xh * w + b
    av = lambda t: t.abs().mean(-1, keepdim=True)  # noqa: E731
    e0 = KS * U * av(x)
    left = KS * U * (av(c) + e0)
    rel = KS * U + left * left / (2 * var) + 4 * U       # of rstd
    exh = rstd * (2 * U * (c.abs() + e0) + 2 * left) + xh.abs() * rel
    ty = w.abs() * exh + 4 * U * (y.abs() + b.abs() + w.abs() * xh.abs())
    gn = gy * w
    m0, m1 = gn.mean(-1, keepdim=True), (gn * xh).mean(-1, keepdim=True)
    gx = rstd * (gn - m0 - xh * m1)
    ex = exh + rstd * U * mean.abs()                     # of xh in the backward pass
    tgx = rstd * (KS * U * (gn.abs() + av(gn) + xh.abs() * av(gn * xh)) + ex * m1.abs()
                  + (xh.abs() + ex) * (gn.abs() * ex).mean(-1, keepdim=True)) + (rel + 4 * U) * gx.abs()
    rows = x.shape[0]
    gw, gb = (gy * xh).sum(0), gy.sum(0)
    tgw = (gy.abs() * ex).sum(0) + (KS + rows) * U * (gy * xh).abs().sum(0)
    tgb = (KS + rows) * U * gy.abs().sum(0)
    return (y, gx, gw, gb), (ty, tgx, tgw, tgb)


def check(x, w, b, gy, eps=1e-5):
    x, w, b = (t.requires_grad_() for t in (x, w, b))
    y = K.layer_norm(x, w, b, eps)
    got = [y, *torch.autograd.grad(y, (x, w, b), gy)]
    with torch.no_grad():
        assert torch.equal(K.layer_norm(x, w, b, eps), y)
    ref, tol = reference(x, w, b, gy, eps)
    for o, r, t, what in zip(got, ref, tol, ("y", "x.grad", "w.grad", "b.grad")):
        d = (wide(o) - r).abs()
        t = t + torch.finfo(o.dtype).eps / 2 * (r.abs() + t)
        assert torch.isfinite(d).all() and (d <= t).all(), (what, (d - t).max().item(), d.max().item())


def inputs(rows, d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    f = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return f, (f(d) * 0.2 + 1).cuda(), (f(d) * 0.2).cuda(), f(rows, d).to(dtype).cuda()


LENGTHS = [3, 7, 40, 47, 200, 255, 768, 1000, 2040, 4095, 6000, 16383]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d", LENGTHS)
def test_constant_rows(d, dtype, device):
    """The bias, whatever the constant: row sums and 1 / d are rounded, their product is
    not the constant."""
    values = torch.tensor([1000.3, -12345.6, 65537.3, 3.0, 1e-3, 0.1, 0.0, -7e4])
    _, w, b, gy = inputs(len(values), d, dtype, d)
    x = values[:, None].expand(-1, d).contiguous().to(dtype).cuda()
    check(x, w, b, gy)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d", LENGTHS)
@pytest.mark.parametrize("spread", [1, 30, 1000])
def test_nearly_constant_rows(d, spread, dtype, device):
    """A few units of the last place around a constant."""
    f, w, b, gy = inputs(6, d, dtype, 7 * d + spread)
    at = torch.tensor([1000.3, -12345.6, 65537.3, 1.7, 5e-4, -7e4]).to(dtype).double()
    step = at.abs().log2().floor().exp2() * torch.finfo(dtype).eps
    k = (f(6, d).double() * spread).round() if spread > 1 else (f(6, d) > 1).double()
    x = (at[:, None] + step[:, None] * k).to(dtype).cuda()
    check(x, w, b, gy)


def test_infinities_and_nan_stay_in_their_rows(device):
    for d in (40, 768, 4095, 5000):
        f, w, b, _ = inputs(5, d, F32, d)
        x = f(5, d).cuda()
        ref = K.layer_norm(x, w, b)
        x[1, d // 2] = float("inf")
        x[3, 0] = float("nan")
        y = K.layer_norm(x, w, b)
        assert y[3].isnan().all() and y[1].isnan().all()
        for i in (0, 2, 4):
            assert torch.equal(y[i], ref[i])

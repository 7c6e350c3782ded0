"""The dense operators (layer norm, fused linear, gated block) against plain
implementations in 64 bits on the same inputs, gradients included.

Tolerances. u = 2^-24 is the rounding of an fp32 operation, half = eps / 2 of the
rows' type. A sum of n products in fp32 is off by at most n u sum|terms|, in any order;
activations and their slopes are off by at most 16 u (1 + |z|) relative to their scale
(a few fp32 operations, one of them an exponential or error function); one rounding to
the rows' type is half of the value. The errors are carried through the formulas with
the magnitudes of what they multiply (bounds below). Besides, the normwise error of a
result that is rounded once is at most half, and half more for each rounded operand.
"""

from __future__ import annotations

import math

import pytest
import torch

from triton_moe import kernels as K

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF16, F32 = torch.bfloat16, torch.float32
f = torch.nn.functional

ACTS = {None: lambda z: z, "relu": torch.relu, "relu_squared": lambda z: torch.relu(z) ** 2,
        "silu": f.silu, "gelu": f.gelu, "gelu_tanh": lambda z: f.gelu(z, approximate="tanh")}
GATES = {"swiglu": "silu", "geglu": "gelu", "geglu_tanh": "gelu_tanh", "reglu": "relu"}


def half(t):
    return torch.finfo(t.dtype).eps / 2


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rnd(g, *shape, dtype=F32, std=1.0, mean=0.0, device="cuda"):
    return (torch.randn(*shape, generator=g) * std + mean).to(dtype).to(device)


def matrix(g, rows, cols, dtype, transposed):
    std = rows ** -0.5
    if transposed:
        return rnd(g, cols, rows, dtype=dtype, std=std).t()
    return rnd(g, rows, cols, dtype=dtype, std=std)


def wide(t):
    return None if t is None else t.detach().cpu().double()


def slope(name, z):
    """The activation's derivative in 64 bits (relu: 0 at 0)."""
    z = z.detach().requires_grad_()
    return torch.autograd.grad(ACTS[name](z).sum(), z)[0]


def close(got, ref, tol, what, rounded=1):
    """|got - ref| <= tol everywhere and rounded * half normwise."""
    assert got.shape == ref.shape, what
    d = (wide(got) - ref).abs()
    assert torch.isfinite(d).all(), what
    over = (d - tol).max().item() if d.numel() else 0.0
    assert over <= 0, f"{what}: {over:.3e} over the bound (largest error {d.max():.3e})"
    norm = ref.norm().item()
    if norm and ref.numel() > 256 and got.dtype == BF16:
        assert d.norm().item() <= rounded * half(got) * norm, what


# ---------------------------------------------------------------------------
# layer norm

NORM_K = 64  # fp32 operations in a row's sums: 16 in a thread, 6 + 16 across, few around


def norm_reference(x, w, b, gy, eps):
    """y, gx, gw, gb in 64 bits and their bounds (without the last rounding)."""
    x, gy = wide(x), wide(gy)
    d, rows = x.shape[-1], x.shape[0]
    w1 = torch.ones(d).double() if w is None else wide(w)
    b0 = torch.zeros(d).double() if b is None else wide(b)
    c = x - x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    xh = c * rstd
    y = xh * w1 + b0
    # what one u does to xh: the mean's and the difference's rounding, and rstd's
    a = rstd * (x.abs() + x.abs().mean(-1, keepdim=True)) + xh.abs() * 2
    ty = NORM_K * U * (w1.abs() * a + b0.abs())
    gn = gy * w1
    m0, m1 = gn.mean(-1, keepdim=True), (gn * xh).mean(-1, keepdim=True)
    gx = rstd * (gn - m0 - xh * m1)
    tgx = NORM_K * U * rstd * (
        2 * gn.abs() + 2 * gn.abs().mean(-1, keepdim=True)
        + 2 * xh.abs() * (gn * xh).abs().mean(-1, keepdim=True)
        + a * m1.abs() + xh.abs() * (gn.abs() * a).mean(-1, keepdim=True)
        + (a * xh.abs()).mean(-1, keepdim=True) * (gn - m0 - xh * m1).abs())
    gw, gb = (gy * xh).sum(0), gy.sum(0)
    chain = NORM_K + rows  # fp32 additions on the way into one sum
    tgw = U * (chain * (gy * xh).abs().sum(0) + NORM_K * (gy.abs() * a).sum(0))
    tgb = U * chain * gy.abs().sum(0)
    return (y, gx, gw, gb), (ty, tgx, tgw, tgb)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,d,wtype", [
    (1, 1, "same"), (3, 2, "same"), (1, 8, "f32"), (5, 17, "none"), (2, 64, "other"),
    (70, 72, "same"), (9, 511, "same"), (33, 512, "f32"), (4, 1000, "other"), (1, 1024, "none"),
    (6, 1025, "same"), (130, 2048, "f32"), (3, 2056, "same"), (7, 4095, "same"), (5, 4096, "same"),
    (3, 5000, "none"), (2, 8193, "same"), (2, 16384, "f32"), (4101, 40, "same"),
    (2500, 260, "none"), (9, 7, "f32"), (300, 47, "same"), (33, 63, "other"), (40, 65, "same"),
    (90, 129, "none"), (21, 255, "same"), (5, 509, "f32"), (3, 2049, "same"), (2, 16383, "same"),
])
def test_layer_norm(rows, d, wtype, dtype, device):
    g = gen(rows * 31 + d)
    eps = 1e-2 if d < 8 else 1e-5
    x = rnd(g, rows, d, dtype=dtype, mean=0.5).requires_grad_()
    gy = rnd(g, rows, d, dtype=dtype)
    wt = {"same": dtype, "f32": F32, "other": BF16 if dtype == F32 else F32, "none": None}[wtype]
    w = b = None
    if wt is not None:
        w = rnd(g, d, dtype=wt, std=0.2, mean=1.0).requires_grad_()
        b = rnd(g, d, dtype=wt, std=0.2).requires_grad_()
    y = K.layer_norm(x, w, b, eps=eps)
    assert y.dtype == dtype
    with torch.no_grad():
        assert torch.equal(K.layer_norm(x, w, b, eps=eps), y)
    leaves = [t for t in (x, w, b) if t is not None]
    got = [y, *torch.autograd.grad(y, leaves, gy)]
    ref, tol = norm_reference(x, w, b, gy, eps)
    for o, r, t, what in zip(got, ref, tol, ("y", "x.grad", "w.grad", "b.grad")):
        close(o, r, t + half(o) * r.abs(), what)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_layer_norm_reads_any_layout(dtype, device):
    """Offsets, row distances and orders give what a contiguous copy gives."""
    g = gen(2)
    base = rnd(g, 41, 300, dtype=dtype)
    w, b = rnd(g, 301, dtype=dtype), rnd(g, 600, dtype=dtype)
    views = [base[:, 1:257], base[::3, :256], base[:, :256].t().contiguous().t(), base[7:8, 3:],
             base[:1].expand(9, 300)[:, :256], base[:, ::2], base.view(41, 3, 100)[:, 1]]
    for v in views:
        d = v.shape[-1]
        for ww, bb in ((None, None), (w[1:d + 1], b[::2][:d]), (w[:d], None), (None, b[3:d + 3])):
            cw, cb = (None if t is None else t.clone() for t in (ww, bb))
            x = v.clone(memory_format=torch.contiguous_format)
            # (A narrower load adds a row's values in another order: each result is
            # within its bound of the 64-bit one, so they are within twice that of each
            # other. The mean's rounding is a share of |x|, not of |y|.)
            (y, *_), (t, *_) = norm_reference(x, cw, cb, x, 1e-5)
            a, c = wide(K.layer_norm(v, ww, bb)), wide(K.layer_norm(x, cw, cb))
            assert ((a - c).abs() <= 2 * (t + half(v) * (y.abs() + t))).all()
    x3 = base.view(41, 3, 100).clone()
    assert torch.equal(K.layer_norm(x3), K.layer_norm(x3.view(-1, 100)).view(41, 3, 100))
    assert torch.equal(K.layer_norm(x3[0, 0]), K.layer_norm(x3.view(-1, 100))[0])


def test_layer_norm_of_special_rows(device):
    """A constant row gives the bias; infinities and NaN stay in their rows; a large
    mean costs no more than its rounding."""
    b = torch.linspace(-1, 1, 256, device="cuda")
    x = rnd(gen(4), 6, 256)
    ref = K.layer_norm(x, None, b)
    x[1] = 3.0
    x[2, 5] = math.inf
    x[4, 200] = math.nan
    y = K.layer_norm(x, None, b)
    assert torch.equal(y[1], b)
    assert y[2].isnan().any() and y[4].isnan().all()
    for i in (0, 3, 5):
        assert torch.equal(y[i], ref[i])
    big = rnd(gen(5), 3, 1000, std=2.0, mean=1000.0)
    (want, *_), (tol, *_) = norm_reference(big, None, None, big, 1e-5)
    close(K.layer_norm(big), want, tol + half(big) * want.abs(), "large mean")


# ---------------------------------------------------------------------------
# products

def act_error(name, z, dz):
    """What an error dz of z, and the fp32 arithmetic, do to the activation."""
    lip = (2 * z.abs() + 2 * dz) if name == "relu_squared" else 1.2
    return lip * dz + 16 * U * (1 + z.abs()) * ACTS[name](z).abs() + 16 * U * z.abs()


def slope_error(name, z, dz):
    """The same for its derivative (relu: it jumps where z may be on either side of 0)."""
    if name is None:
        return torch.zeros_like(z)
    if name == "relu":
        return (z.abs() <= dz).double()
    return 2 * dz + 16 * U * (1 + z.abs()) * (1 + z.abs())


def linear_reference(x, w, b, r, gy, act):
    x64, w64, b64, r64, g64 = (wide(t) for t in (x, w, b, r, gy))
    hx = half(x) if x.dtype == BF16 else 0.0  # operands rounded to bf16
    rows, k = x64.shape
    n = w64.shape[1]
    z, mag = x64 @ w64, x64.abs() @ w64.abs()
    if b64 is not None:
        z, mag = z + b64, mag + b64.abs()
    dz = (k + 8) * U * mag
    y = ACTS[act](z)
    ty = act_error(act, z, dz)
    if r64 is not None:
        y, ty = y + r64, ty + 2 * U * (y.abs() + r64.abs())
    s, ds = slope(act, z), slope_error(act, z, dz)
    gz, tgz = g64 * s, g64.abs() * (ds + 2 * U * s.abs())
    rounded = tgz + (hx if act else 0.0) * (gz.abs() + tgz)  # the products' operand
    gx, gw, gb = gz @ w64.t(), x64.t() @ gz, gz.sum(0)
    tgx = rounded @ w64.abs().t() + (n + 8) * U * (gz.abs() @ w64.abs().t())
    tgw = x64.abs().t() @ rounded + (rows + 8) * U * (x64.abs().t() @ gz.abs())
    tgb = tgz.sum(0) + (rows + 8) * U * gz.abs().sum(0)
    return (y, gx, gw, gb), (ty, tgx, tgw, tgb)


ROWS_IN_OUT = [
    (1, 8, 8), (1, 64, 136), (1, 2056, 72), (3, 40, 72), (7, 1032, 264), (16, 520, 264),
    (17, 72, 1032), (32, 2048, 40), (33, 264, 520), (61, 1032, 136), (64, 2056, 264),
    (65, 136, 264), (130, 520, 392), (257, 72, 520), (300, 4096, 264), (1100, 264, 1032),
    (2051, 72, 776),
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("i", range(len(ROWS_IN_OUT)))
def test_fused_linear(i, dtype, device):
    rows, k, n = ROWS_IN_OUT[i]
    acts = list(ACTS)
    for transposed in (False, True):
        act = acts[(i + 3 * transposed) % len(acts)]
        use_b, use_r = bool((i + transposed) & 1), bool((i + transposed) & 2) or i == 0
        g = gen(100 * i + transposed)
        x = rnd(g, rows, k, dtype=dtype).requires_grad_()
        w = matrix(g, k, n, dtype, transposed).requires_grad_()
        bt = dtype if i % 3 else F32
        b = rnd(g, n, dtype=bt, std=0.5).requires_grad_() if use_b else None
        r = rnd(g, rows, n, dtype=dtype).requires_grad_() if use_r else None
        gy = rnd(g, rows, n, dtype=dtype)
        y = K.fused_linear(x, w, b, act, r)
        with torch.no_grad():
            assert torch.equal(K.fused_linear(x, w, b, act, r), y)
        leaves = [t for t in (x, w, b, r) if t is not None]
        grads = dict(zip(("x", "w", *(["b"] if use_b else []), *(["r"] if use_r else [])),
                         torch.autograd.grad(y, leaves, gy)))
        assert grads["w"].stride() == w.stride()
        (ry, rx, rw, rb), (ty, tx, tw, tb) = linear_reference(x, w, b, r, gy, act)
        what = f"{act} transposed {transposed} "
        close(y, ry, ty + half(y) * (ry.abs() + ty), what + "y")
        close(grads["x"], rx, tx + half(x) * (rx.abs() + tx), what + "x.grad", 2)
        close(grads["w"], rw, tw + half(w) * (rw.abs() + tw), what + "w.grad", 2)
        if use_b:
            assert grads["b"].dtype == bt
            close(grads["b"], rb, tb + half(b) * (rb.abs() + tb), what + "b.grad")
        if use_r:
            assert torch.equal(grads["r"], gy)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("act", list(ACTS))
def test_activations_over_their_range(act, dtype, device):
    """Arguments from tiny to saturated, of both signs, through a unit weight."""
    v = torch.cat([torch.linspace(-30, 30, 1003), torch.tensor([0.0, -0.0, 1e-6, -1e-6, 90.0, -90.0,
                                                               200.0, -200.0, 1e4, -1e4, 3e9])])
    n = 8
    x = torch.zeros(v.numel(), 8)
    x[:, 0] = v
    x = x.to(dtype).cuda().requires_grad_()
    w = torch.zeros(8, n, device="cuda", dtype=dtype)
    w[0] = 1.0
    gy = torch.ones(v.numel(), n, device="cuda", dtype=dtype) / 8
    y = K.fused_linear(x, w, None, act)
    gx, = torch.autograd.grad(y, x, gy)
    z = wide(x)[:, :1]
    ref = ACTS[act](z).expand(-1, n)
    close(y, ref, (half(y) * ref.abs() + 16 * U * ((1 + z.abs()) * ref.abs() + z.abs()))
          .expand(-1, n), "y")
    # the row's gradient: the sum over n of gy slope, each rounded
    s = slope(act, z)
    ref = torch.zeros_like(wide(x))
    ref[:, :1] = s
    tol = torch.zeros_like(ref)
    tol[:, :1] = 2 * half(x) * s.abs() + (0 if act in (None, "relu")
                                          else 32 * U * (1 + z.abs()) * (1 + z.abs()))
    close(gx, ref, tol, "x.grad", 2)


def gated_reference(x, w1, w2, b1, b2, r, gy, act):
    act = GATES[act]
    x64, w164, w264, b164, b264, r64, g64 = (wide(t) for t in (x, w1, w2, b1, b2, r, gy))
    hx = half(x) if x.dtype == BF16 else 0.0
    rows, d = x64.shape
    width = w264.shape[0]
    z, mag = x64 @ w164, x64.abs() @ w164.abs()
    if b164 is not None:
        z, mag = z + b164, mag + b164.abs()
    dz = (d + 8) * U * mag
    (zg, zu), (eg, eu) = z.chunk(2, 1), dz.chunk(2, 1)
    a, ta = ACTS[act](zg), act_error(act, zg, eg)
    h = a * zu
    th = ta * (zu.abs() + eu) + a.abs() * eu + 2 * U * h.abs()
    rh = th + hx * (h.abs() + th)  # rounded: the second product's operand
    y = h @ w264
    ty = rh @ w264.abs() + (width + 8) * U * (h.abs() @ w264.abs())
    for t in (b264, r64):
        if t is not None:
            y, ty = y + t, ty + 2 * U * (y.abs() + t.abs())
    gh = g64 @ w264.t()
    tgh = (d + 8) * U * (g64.abs() @ w264.abs().t())
    s, ds = slope(act, zg), slope_error(act, zg, eg)
    gg, gu = gh * zu * s, gh * a
    tgg = tgh * (zu.abs() * s.abs()) + (gh.abs() + tgh) * (eu * s.abs() + (zu.abs() + eu) * ds) \
        + 4 * U * gg.abs()
    tgu = tgh * a.abs() + (gh.abs() + tgh) * ta + 2 * U * gu.abs()
    gz, tgz = torch.cat([gg, gu], 1), torch.cat([tgg, tgu], 1)
    rgz = tgz + hx * (gz.abs() + tgz)
    gx = gz @ w164.t()
    tgx = rgz @ w164.abs().t() + (2 * width + 8) * U * (gz.abs() @ w164.abs().t())
    gw1 = x64.t() @ gz
    tgw1 = x64.abs().t() @ rgz + (rows + 8) * U * (x64.abs().t() @ gz.abs())
    gw2 = h.t() @ g64
    tgw2 = rh.t() @ g64.abs() + (rows + 8) * U * (h.abs().t() @ g64.abs())
    gb1, gb2 = gz.sum(0), g64.sum(0)
    tgb1 = tgz.sum(0) + (rows + 8) * U * gz.abs().sum(0)
    tgb2 = (rows + 8) * U * g64.abs().sum(0)
    return (y, gx, gw1, gw2, gb1, gb2), (ty, tgx, tgw1, tgw2, tgb1, tgb2)


ROWS_D_WIDTH = [
    (1, 8, 8), (1, 64, 200), (2, 1032, 72), (16, 264, 520), (17, 136, 40), (31, 72, 1032),
    (33, 2056, 136), (64, 264, 264), (65, 520, 72), (129, 72, 264), (300, 264, 520),
    (700, 1536, 136), (2051, 136, 264),
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("i", range(len(ROWS_D_WIDTH)))
def test_gated_mlp(i, dtype, device):
    rows, d, width = ROWS_D_WIDTH[i]
    for t in (0, 1):
        act = sorted(GATES)[(i + 2 * t) % 4]
        t1, t2 = bool((i + t) & 1), bool((i >> 1) + t & 1)
        use_b, use_r = bool((i + t) % 3), bool((i + t) & 1)
        g = gen(1000 + 10 * i + t)
        x = rnd(g, rows, d, dtype=dtype).requires_grad_()
        w1 = matrix(g, d, 2 * width, dtype, t1).requires_grad_()
        w2 = matrix(g, width, d, dtype, t2).requires_grad_()
        b1 = rnd(g, 2 * width, dtype=dtype, std=0.5).requires_grad_() if use_b else None
        b2 = rnd(g, d, dtype=F32, std=0.5).requires_grad_() if use_b else None
        r = rnd(g, rows, d, dtype=dtype).requires_grad_() if use_r else None
        gy = rnd(g, rows, d, dtype=dtype)
        y = K.gated_mlp(x, w1, w2, act, b1, b2, r)
        with torch.no_grad():
            assert torch.equal(K.gated_mlp(x, w1, w2, act, b1, b2, r), y)
        named = [(n, v) for n, v in zip(("x", "w1", "w2", "b1", "b2", "r"),
                                        (x, w1, w2, b1, b2, r)) if v is not None]
        grads = dict(zip([n for n, _ in named],
                         torch.autograd.grad(y, [v for _, v in named], gy)))
        ref, tol = gated_reference(x, w1, w2, b1, b2, r, gy, act)
        what = f"{act} {t1} {t2} "
        close(y, ref[0], tol[0] + half(y) * (ref[0].abs() + tol[0]), what + "y", 2)
        for n, v, q in zip(("x", "w1", "w2", "b1", "b2"), ref[1:], tol[1:]):
            if n in grads:
                o = grads[n]
                close(o, v, q + half(o) * (v.abs() + q), what + n + ".grad", 2)
                assert o.stride() == dict(named)[n].stride()
        if use_r:
            assert torch.equal(grads["r"], gy)


def test_tiles_of_every_size(device):
    """Products that fill the card with the largest tiles, with a partial tile at each
    edge and a tail of tiles split along k: against the same rows, a few at a time and
    in fp32 from the same values (rounded once each)."""
    g = gen(9)
    for rows, k, n in ((4099, 72, 4104), (5000, 520, 1032), (1500, 1032, 2056)):
        x = rnd(g, rows, k, dtype=BF16).requires_grad_()
        for transposed in (False, True):
            w = matrix(g, k, n, BF16, transposed).requires_grad_()
            gy = rnd(g, rows, n, dtype=BF16)
            y = K.fused_linear(x, w)
            gx, gw = torch.autograd.grad(y, (x, w), gy)
            x64, w64, g64 = (t.detach().double() for t in (x, w, gy))
            for got, a, b, terms in ((y, x64, w64, k), (gx, g64, w64.t().contiguous(), n),
                                     (gw, x64.t().contiguous(), g64, rows)):
                ref = a.matmul(b)
                tol = half(got) * ref.abs() + 2 * (terms + 8) * U * a.abs().matmul(b.abs())
                assert ((got.double() - ref).abs() <= tol).all(), (rows, k, n, transposed)
    rows, d, width = 4099, 136, 2056
    x = rnd(g, rows, d, dtype=BF16).requires_grad_()
    w1, w2 = matrix(g, d, 2 * width, BF16, False), matrix(g, width, d, BF16, False)
    w1.requires_grad_()
    b1 = rnd(g, 2 * width, dtype=BF16).requires_grad_()
    w2.requires_grad_()
    gy = rnd(g, rows, d, dtype=BF16)
    y = K.gated_mlp(x, w1, w2, "swiglu", b1)
    got = [y, *torch.autograd.grad(y, (x, w1, w2, b1), gy)]
    ref, tol = gated_reference(x, w1, w2, b1, None, None, gy, "swiglu")
    for o, v, q, what in zip(got, ref, tol, ("y", "x", "w1", "w2", "b1")):
        close(o, v, q + half(o) * (v.abs() + q), what, 2)


def test_rows_do_not_touch_each_other(device):
    """Infinities and NaN of one row leave the others' bits alone, at sizes that end
    inside a tile."""
    for rows, k, n, dtype in ((5, 72, 40, BF16), (70, 264, 136, BF16), (130, 40, 68, F32),
                              (300, 4096, 264, BF16)):
        g = gen(rows)
        x = rnd(g, rows, k, dtype=dtype)
        w1, w2 = matrix(g, k, 2 * n, dtype, False), matrix(g, n, k, dtype, True)
        w = matrix(g, k, n, dtype, True)
        y, z = K.fused_linear(x, w, activation="gelu"), K.gated_mlp(x, w1, w2)
        x2 = x.clone()
        x2[rows // 2] = math.nan
        x2[-1, 0] = math.inf
        y2, z2 = K.fused_linear(x2, w, activation="gelu"), K.gated_mlp(x2, w1, w2)
        keep = [i for i in range(rows - 1) if i != rows // 2]
        assert torch.equal(y[keep], y2[keep]) and torch.equal(z[keep], z2[keep])
        assert y2[rows // 2].isnan().all() and z2[rows // 2].isnan().all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_products_read_any_layout(dtype, device):
    """Row distances, offsets and orders that the kernels do not read in place are
    copied: the bits of contiguous inputs."""
    g = gen(11)
    k, n = 72, 136
    base = rnd(g, 40, 3 * k, dtype=dtype)
    wide_w = rnd(g, k + 3, 2 * n + 16, dtype=dtype, std=0.1)
    views_x = [base[:, :k], base[:, 1:k + 1], base[::2, k:2 * k], base[:, ::3],
               base[:, :k].t().contiguous().t(), base[3:4, 5:k + 5], base[:1, :k].expand(6, k),
               base[:32, :k].reshape(2, 4, 4, k), base[0, :k]]
    views_w = [wide_w[:k, :n], wide_w[1:k + 1, 3:n + 3], wide_w[:k, ::2][:, :n],
               rnd(g, n, k + 8, dtype=dtype, std=0.1)[:, :k].t(),
               rnd(g, n, k + 3, dtype=dtype, std=0.1)[:, 3:].t()]
    for v in views_x:
        for w in views_w:
            r = rnd(g, n + 1, *v.shape[:-1], dtype=dtype)[1:].movedim(0, -1)
            b = rnd(g, 2 * n, dtype=dtype)[::2]
            got = K.fused_linear(v, w, b, "silu", r)
            order = w.t().clone(memory_format=torch.contiguous_format).t() if w.stride(0) == 1 \
                else w.clone(memory_format=torch.contiguous_format)
            want = K.fused_linear(v.clone(memory_format=torch.contiguous_format), order, b.clone(),
                                  "silu", r.clone(memory_format=torch.contiguous_format))
            assert got.is_contiguous() and torch.equal(got, want)
    # gradients of broadcast rows, and a gradient with no distance between rows
    x = base[:1, :k].clone().requires_grad_()
    w = wide_w[:k, :n].clone().requires_grad_()
    y = K.fused_linear(x.expand(6, k), w)
    y.sum().backward()
    one = rnd(g, 1, 1, dtype=dtype) * 0 + 1
    gx, = torch.autograd.grad(K.fused_linear(x, w), x, one.expand(1, n))
    # torch adds the six rows' gradients one by one: 2 g, 3 g, ... 6 g are rounded, half
    # of 20 g together; one row and six may sum in other orders (bound of a product)
    close(x.grad, 6 * wide(gx), 20 * half(x) * wide(gx).abs() +
          12 * (n + 8) * U * wide(w).abs().sum(1), "broadcast rows")


def test_weight_at_an_address_that_is_not_aligned(device):
    g = gen(12)
    flat = rnd(g, 64 * 64 + 1, dtype=BF16)
    w = flat[1:].view(64, 64)
    x = rnd(g, 9, 64, dtype=BF16)
    assert w.data_ptr() % 16 and torch.equal(K.fused_linear(x, w), K.fused_linear(x, w.clone()))
    assert torch.equal(K.gated_mlp(x, w, w[:32]), K.gated_mlp(x, w.clone(), w[:32].clone()))
    assert torch.equal(K.fused_linear(x, w.t()), K.fused_linear(x, w.t().clone().t().t()
                                                               .t().contiguous().t()))


def test_negative_views(device):
    g = gen(18)
    x, w, b = rnd(g, 9, 64), rnd(g, 64, 64), rnd(g, 64)
    nx, nw, nb = (torch.complex(torch.zeros_like(t), -t).conj().imag for t in (x, w, b))
    assert nx.is_neg() and torch.equal(nx, x)
    assert torch.equal(K.layer_norm(nx, nb, nb), K.layer_norm(x, b, b))
    assert torch.equal(K.fused_linear(nx, nw, nb, "gelu", nx), K.fused_linear(x, w, b, "gelu", x))
    assert torch.equal(K.gated_mlp(nx, nw, nw[:32], "reglu", nb, nb, nx),
                       K.gated_mlp(x, w, w[:32], "reglu", b, b, x))


def test_offsets_past_32_bits(device):
    """Rows behind the first 4 GiB, and 2^31 values, of inputs and outputs."""
    rows, d = 300_000, 8192
    x = torch.zeros(rows, d, device="cuda", dtype=BF16)
    g = gen(19)
    at = [0, 1, 131_071, 131_072, 262_143, 262_144, 262_145, rows - 1]
    values = rnd(g, len(at), d, dtype=BF16)
    x[at] = values
    y = K.layer_norm(x)
    (want, *_), (t, *_) = norm_reference(values, None, None, values, 1e-5)
    close(y[at], want, t + half(x) * want.abs(), "layer_norm")
    assert not y[5].any() and not y[rows - 2].any()
    del y
    for n in (8, 264):
        w = matrix(g, d, n, BF16, n == 8)
        y = K.fused_linear(x, w)
        (want, *_), (t, *_) = linear_reference(values, w, None, None, rnd(g, len(at), n, dtype=BF16),
                                               None)
        close(y[at], want, t + half(x) * (want.abs() + t), f"fused_linear {n}")
        assert not y[rows - 2].any()
    w = matrix(g, 8, d, BF16, False)  # a long output
    y = K.fused_linear(x[:, :8], w, residual=x)
    (want, *_), (t, *_) = linear_reference(values[:, :8], w, None, values, values, None)
    close(y[at], want, t + half(x) * (want.abs() + t), "long output")
    assert not y[rows - 2].any()


def test_no_rows(device):
    w1 = torch.ones(16, 64, device="cuda", requires_grad=True)
    w2 = torch.ones(32, 16, device="cuda", requires_grad=True)
    b1, b2 = (torch.ones(n, device="cuda", requires_grad=True) for n in (64, 16))
    nw = torch.ones(16, device="cuda", requires_grad=True)
    for shape in ((0, 16), (3, 0, 16)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        y = K.gated_mlp(K.layer_norm(x, nw, b2), w1, w2, "geglu", b1, b2, x)
        z = K.fused_linear(x, w1, b1, "gelu")
        assert y.shape == x.shape and z.shape == (*shape[:-1], 64)
        for t in torch.autograd.grad(y.sum() + z.sum(), (x, w1, w2, b1, b2, nw)):
            assert t.numel() == 0 or (t == 0).all()


# ---------------------------------------------------------------------------
# together, and around the calls

def block(p, x, y_of=K):
    """A pre-norm block: a projection with its activation, and a gated block."""
    h = y_of.fused_linear(y_of.layer_norm(x, p["n1"], p["c1"]), p["w"], p["b"], "gelu", x)
    return y_of.gated_mlp(y_of.layer_norm(h, p["n2"], p["c2"]), p["w1"], p["w2"], "swiglu", None,
                          p["b2"], h)


class Plain:
    """The operators in plain torch."""

    @staticmethod
    def layer_norm(x, w, b):
        return f.layer_norm(x, x.shape[-1:], w, b, 1e-5)

    @staticmethod
    def fused_linear(x, w, b, act, r):
        return ACTS[act](x.matmul(w) + b) + r

    @staticmethod
    def gated_mlp(x, w1, w2, act, b1, b2, r):
        g, u = x.matmul(w1).chunk(2, -1)
        return (ACTS[GATES[act]](g) * u).matmul(w2) + b2 + r


def block_params(dtype, d=264, width=520, seed=21):
    g = gen(seed)
    p = dict(n1=rnd(g, d, mean=1.0, std=0.1), c1=rnd(g, d, std=0.1), n2=rnd(g, d, mean=1.0, std=0.1),
             c2=rnd(g, d, std=0.1), w=matrix(g, d, d, dtype, True), b=rnd(g, d, dtype=dtype),
             w1=matrix(g, d, 2 * width, dtype, True), w2=matrix(g, width, d, dtype, False),
             b2=rnd(g, d, dtype=dtype))
    return {k: v.requires_grad_() for k, v in p.items()}


def block_grads(p, x, gy):
    y = block(p, x)
    return [y, *torch.autograd.grad(y, [x, *p.values()], gy)]


@pytest.mark.parametrize("rows", [(1,), (2, 37), (900,)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_block(rows, dtype, device):
    """The operators as they are used, against the same block in 64 bits. bf16 rounds
    at nine places on the way to a gradient; their errors add as squares at best and
    linearly at worst: nine halves, doubled by the residual sums that cancel. fp32: as
    many sums of up to 1040 terms."""
    p = block_params(dtype)
    g = gen(5)
    x = rnd(g, *rows, 264, dtype=dtype).requires_grad_()
    gy = rnd(g, *rows, 264, dtype=dtype)
    got = block_grads(p, x, gy)
    q = {k: wide(v).requires_grad_() for k, v in p.items()}
    x64 = wide(x).requires_grad_()
    y = block(q, x64, Plain)
    ref = [y, *torch.autograd.grad(y, [x64, *q.values()], wide(gy))]
    tol = 18 * 2.0 ** -8 / math.sqrt(3) if dtype == BF16 else 18 * math.sqrt(1040) * U
    for o, r, what in zip(got, ref, ("y", "x", *p)):
        err = (wide(o) - r.detach()).norm() / r.detach().norm()
        assert err <= tol, (what, err)


@pytest.mark.parametrize("op", ["norm", "linear", "gated"])
def test_gradients_against_differences(op, device):
    """Directional derivatives of the plain form in 64 bits by central differences
    (step 1e-4: off by about 1e-8) against the kernels' gradients in fp32: sums of at
    most 2100 products."""
    g = gen(31)
    x = rnd(g, 37, 72).requires_grad_()
    gy = rnd(g, 37, 72)
    if op == "norm":
        ins = [x, rnd(g, 72, mean=1.0).requires_grad_(), rnd(g, 72).requires_grad_()]
        run, plain = K.layer_norm, Plain.layer_norm
    elif op == "linear":
        ins = [x, matrix(g, 72, 72, F32, True).requires_grad_(), rnd(g, 72).requires_grad_(),
               rnd(g, 37, 72).requires_grad_()]
        run = lambda a, w, b, r: K.fused_linear(a, w, b, "gelu_tanh", r)  # noqa: E731
        plain = lambda a, w, b, r: Plain.fused_linear(a, w, b, "gelu_tanh", r)  # noqa: E731
    else:
        ins = [x, matrix(g, 72, 272, F32, False).requires_grad_(),
               matrix(g, 136, 72, F32, True).requires_grad_(), rnd(g, 72).requires_grad_(),
               rnd(g, 37, 72).requires_grad_()]
        run = lambda a, w1, w2, b, r: K.gated_mlp(a, w1, w2, "swiglu", None, b, r)  # noqa: E731
        plain = lambda a, w1, w2, b, r: Plain.gated_mlp(a, w1, w2, "swiglu", None, b, r)  # noqa: E731
    grads = torch.autograd.grad(run(*ins), ins, gy)
    at = [wide(t) for t in ins]
    for i, (t, gr) in enumerate(zip(at, grads)):
        v = torch.randn(t.shape, generator=g).double()
        h = 1e-4
        ends = [(plain(*[a + s * h * v if j == i else a for j, a in enumerate(at)]) * wide(gy)).sum()
                for s in (1, -1)]
        want = (ends[0] - ends[1]) / (2 * h)
        size = (wide(gr).abs() * v.abs()).sum()
        assert abs((wide(gr) * v).sum() - want) <= 2100 * U * size + 1e-6 * size, i


def test_some_gradients(device):
    """Only what is asked for comes back, with the bits of the whole pass; a tensor in
    two places gets both gradients."""
    p = block_params(BF16)
    g = gen(6)
    x = rnd(g, 130, 264, dtype=BF16).requires_grad_()
    gy = rnd(g, 130, 264, dtype=BF16)
    args = (x, p["w1"], p["w2"], "swiglu", None, p["b2"])
    all_ = torch.autograd.grad(K.gated_mlp(*args), (x, p["w1"], p["w2"], p["b2"]), gy)
    for i, t in enumerate((x, p["w1"], p["w2"], p["b2"])):
        assert torch.equal(torch.autograd.grad(K.gated_mlp(*args), t, gy)[0], all_[i])
        others = [v.detach() if v is not t and isinstance(v, torch.Tensor) else v for v in args]
        assert torch.equal(torch.autograd.grad(K.gated_mlp(*others), t, gy)[0], all_[i])
    both, = torch.autograd.grad(K.gated_mlp(*args, x), x, gy)
    assert torch.equal(both, (all_[0].float() + gy.float()).to(BF16))
    for i, t in enumerate((x, p["w"], p["b"])):
        y = K.fused_linear(x, p["w"], p["b"], "silu")
        whole = torch.autograd.grad(y, (x, p["w"], p["b"]), gy, retain_graph=True)
        assert torch.equal(torch.autograd.grad(y, t, gy)[0], whole[i])
    for i, t in enumerate((x, p["n1"], p["c1"])):
        y = K.layer_norm(x, p["n1"], p["c1"])
        whole = torch.autograd.grad(y, (x, p["n1"], p["c1"]), gy, retain_graph=True)
        assert torch.equal(torch.autograd.grad(y, t, gy)[0], whole[i])
    r = rnd(g, 130, 264, dtype=BF16).requires_grad_()  # the residual alone
    for y in (K.fused_linear(x.detach(), p["w"].detach(), residual=r),
              K.gated_mlp(x.detach(), p["w1"].detach(), p["w2"].detach(), residual=r)):
        assert torch.equal(torch.autograd.grad(y, r, gy)[0], gy)


def test_gradients_are_not_differentiated_again(device):
    p = block_params(F32)
    x = rnd(gen(7), 9, 264).requires_grad_()
    for y in (K.layer_norm(x, p["n1"]), K.fused_linear(x, p["w"], p["b"], "silu"),
              K.gated_mlp(x, p["w1"], p["w2"])):
        gx, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="cannot be differentiated again"):
            gx.sum().backward()


def test_forward_mode_is_refused(device):
    import torch.autograd.forward_ad as fwad
    x, w = rnd(gen(8), 3, 16), rnd(gen(9), 16, 16)
    with fwad.dual_level():
        d = fwad.make_dual(x, torch.ones_like(x))
        for call in (lambda: K.layer_norm(d), lambda: K.fused_linear(d, w),
                     lambda: K.fused_linear(x, w, residual=d), lambda: K.gated_mlp(d, w, w[:8])):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_replaced_values_are_refused_in_the_backward_pass(device):
    p = block_params(F32)
    x = rnd(gen(7), 9, 264).requires_grad_()
    for act, residual, kept in (("relu", None, True), ("relu_squared", None, False),
                                ("relu", x, False), ("silu", None, False)):
        y = K.fused_linear(x, p["w"], activation=act, residual=residual)
        y.mul_(2)
        if kept:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                y.sum().backward()
        else:
            y.sum().backward()
    y = K.fused_linear(x, p["w"], activation="gelu")
    with torch.no_grad():
        p["w"].mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("rows", [3, 700])
def test_calls_repeat_their_bits(rows, device):
    p = block_params(BF16)
    g = gen(13)
    x = rnd(g, rows, 264, dtype=BF16).requires_grad_()
    gy = rnd(g, rows, 264, dtype=BF16)
    first = block_grads(p, x, gy)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, block_grads(p, x, gy)))


@pytest.mark.parametrize("rows", [1, 300])
def test_captured_step(rows, device):
    """Forward and backward in a graph, replayed with other values between eager work:
    each replay has the eager step's bits."""
    p = block_params(BF16)
    g = gen(14)
    x = rnd(g, rows, 264, dtype=BF16).requires_grad_()
    gy = rnd(g, rows, 264, dtype=BF16)
    values = [rnd(g, rows, 264, dtype=BF16) for _ in range(3)]
    want = []
    for v in values:
        with torch.no_grad():
            x.copy_(v)
        want.append([t.detach().clone() for t in block_grads(p, x, gy)])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block_grads(p, x, gy)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block_grads(p, x, gy)
    for i in (0, 1, 2, 1, 0):
        with torch.no_grad():
            x.copy_(values[i])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i])), i
        with torch.no_grad():
            block(p, x)
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_few_rows_joined_in_their_launch(dtype, device):
    """Products of few rows that are split along k: joined by the last workgroup of the
    launch in eager calls, by a launch of their own in a graph, with the same bits, again
    and again, and on two streams at once."""
    g = gen(20)
    calls = []
    for rows, k, n in ((1, 2048, 2048), (5, 4104, 72), (23, 4096, 264), (61, 2056, 136), (64, 5632, 8),
                       (17, 1544, 2504)):
        for transposed in (False, True):
            x, w = rnd(g, rows, k, dtype=dtype), matrix(g, k, n, dtype, transposed)
            b, r = rnd(g, n, dtype=dtype), rnd(g, rows, n, dtype=dtype)
            (want, *_), (t, *_) = linear_reference(x, w, b, r, r, "silu")
            y = K.fused_linear(x, w, b, "silu", r)
            close(y, want, t + half(y) * (want.abs() + t), f"{rows} {k} {n} {transposed}")
            calls.append(lambda x=x, w=w, b=b, r=r: K.fused_linear(x, w, b, "silu", r))
    for rows, d, width in ((1, 2056, 2600), (30, 1544, 2056)):
        for transposed in (False, True):
            x, w1 = rnd(g, rows, d, dtype=dtype), matrix(g, d, 2 * width, dtype, transposed)
            w2 = matrix(g, width, d, dtype, not transposed)
            (want, *_), (t, *_) = gated_reference(x, w1, w2, None, None, x, x, "geglu")
            y = K.gated_mlp(x, w1, w2, "geglu", None, None, x)
            close(y, want, t + half(y) * (want.abs() + t), f"gated {rows} {transposed}", 2)
            calls.append(lambda x=x, w1=w1, w2=w2: K.gated_mlp(x, w1, w2, "geglu", None, None, x))
    want = [c() for c in calls]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = [c() for c in calls]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got.append([c() for c in calls])
        graph.replay()
        torch.cuda.synchronize()
        for ys in (*got, captured):
            assert all(torch.equal(a, b) for a, b in zip(ys, want))


def test_inference_mode_first(device):
    """What a stream keeps is made in inference mode and used outside of it."""
    g = gen(22)
    x, w = rnd(g, 2, 4096, dtype=BF16), matrix(g, 4096, 64, BF16, False).requires_grad_()
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
        with torch.inference_mode():
            a = K.fused_linear(x, w)
        b = K.fused_linear(x, w)
        b.sum().backward()
    torch.cuda.synchronize()
    assert a.is_inference() and torch.equal(a, b) and w.grad is not None


def test_two_streams_at_once(device):
    """Calls on two streams share nothing."""
    p = block_params(BF16)
    g = gen(15)
    xs = [rnd(g, n, 264, dtype=BF16).requires_grad_() for n in (300, 517)]
    gys = [torch.ones_like(x) for x in xs]
    want = [block_grads(p, x, gy) for x, gy in zip(xs, gys)]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(block_grads(p, xs[i], gys[i]))
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        for r in runs:
            assert all(torch.equal(a, b) for a, b in zip(w, r))


def test_compiled_caller(device):
    p = block_params(BF16)
    x = rnd(gen(16), 40, 264, dtype=BF16)
    with torch.no_grad():
        want = block(p, x)
        torch.compiler.reset()
        got = torch.compile(lambda t: block(p, t) + 0, backend="eager")(x)
        torch.compiler.reset()
    assert torch.equal(got, want)


def test_launch_observer(device):
    from triton_moe import _lib

    class Timer:
        def __init__(self):
            self.seen = []

        def begin(self, name):
            self.seen.append(("begin", name))

        def end(self, name):
            self.seen.append(("end", name))

    t = Timer()
    x = rnd(gen(17), 4, 64).requires_grad_()
    _lib.dense()
    _lib.set_launch_timer(t)
    try:
        K.layer_norm(x).sum().backward()
    finally:
        _lib.set_launch_timer(None)
    assert t.seen == [(w, n) for n in ("vmoe_layer_norm", "vmoe_layer_norm_backward")
                      for w in ("begin", "end")]
    K.layer_norm(x)
    assert len(t.seen) == 4

"""Every kernel that the dense operators can take, whole, split along k and with both
kinds of tiles in one product, at sizes that end inside tiles and stages, against the
64-bit references of test_gpu_dense.py and with its bounds; and the launch rules of
_dense_variants.py against the kernels that run."""

from __future__ import annotations

from functools import partial

import pytest
import torch
from torch.profiler import ProfilerActivity, profile

import _dense_variants as V
import test_gpu_dense as dense
from test_gpu_dense import BF16, F32, GATES, close, gated_reference, gen, half, linear_reference, \
    matrix, norm_reference, rnd
from triton_moe import kernels as K

pytestmark = pytest.mark.gpu

DTYPE = {"bf16": BF16, "f32": F32}

LINEAR = [
    # type, rows, in, out, weight stored [out, in], activation, bias, residual, what runs
    # (train: both passes; graph: the forward pass alone, in a graph)
    ("bf16", 1, 1032, 8, True, "gelu", True, False, "graph"),
    ("bf16", 1, 1096, 8, False, "gelu", True, True, "graph"),
    ("bf16", 19, 1048, 8, False, "gelu_tanh", True, False, "graph"),
    ("bf16", 35, 1056, 72, False, "relu", False, False, "graph"),
    ("bf16", 5556, 5104, 648, True, "gelu", False, False, "train"),
    ("bf16", 4515, 4072, 3344, False, "relu", True, False, "train"),
    ("bf16", 8227, 136, 2056, False, "silu", True, False, "train"),      # z past the caches
    ("bf16", 8227, 72, 2056, True, "relu", True, True, "train"),
    ("bf16", 2, 488, 12936, False, "silu", True, True, "train"),          # 64 columns, whole
    ("bf16", 17, 432, 14584, False, "gelu", False, True, "train"),
    ("bf16", 37, 456, 13816, False, None, True, False, "train"),
    ("bf16", 1, 1976, 3192, False, "relu", False, False, "graph"),        # 64 columns, split
    ("bf16", 17, 2496, 2536, False, "gelu_tanh", True, False, "train"),
    ("bf16", 35, 2752, 2296, False, None, True, True, "graph"),
    ("f32", 1, 1132, 8, False, "relu_squared", True, True, "graph"),
    ("f32", 1, 1144, 8, True, "gelu_tanh", False, True, "graph"),
    ("f32", 33, 1084, 8, True, None, False, True, "graph"),
    ("f32", 37, 1320, 72, False, "gelu", True, False, "graph"),
    ("f32", 33, 1104, 12, False, "silu", False, False, "train"),
    ("f32", 1375, 3796, 524, False, "relu", True, False, "train"),
    ("f32", 8227, 68, 2052, True, "gelu", True, False, "train"),         # z past the caches
]

GATED = [
    # type, rows, d, width, w1 and w2 stored [out, in], biases, what runs
    ("bf16", 1, 8, 8, True, False, False, "graph"),
    ("bf16", 1, 8, 8, False, True, True, "graph"),
    ("bf16", 17, 8, 8, True, True, False, "graph"),
    ("bf16", 18, 8, 8, False, False, True, "graph"),
    ("bf16", 34, 8, 8, False, True, False, "graph"),
    ("bf16", 65, 8, 8, True, False, True, "train"),
    ("bf16", 66, 8, 8, False, False, True, "train"),
    ("bf16", 1, 1040, 8, False, True, True, "train"),
    ("bf16", 17, 1056, 8, False, False, True, "train"),
    ("bf16", 73, 456, 8, True, False, True, "train"),
    ("bf16", 33, 1152, 8, True, False, True, "train"),
    ("bf16", 42, 1080, 8, False, False, False, "train"),
    ("bf16", 1, 3160, 1000, False, True, False, "graph"),
    ("bf16", 1, 1120, 2832, False, False, True, "graph"),
    ("bf16", 4, 3440, 1000, True, False, True, "train"),
    ("bf16", 17, 2008, 1600, False, True, True, "graph"),
    ("bf16", 35, 904, 3528, False, True, True, "graph"),
    ("bf16", 18, 3888, 864, True, True, False, "train"),
    ("bf16", 17, 1424, 2984, False, False, True, "train"),
    ("bf16", 38, 3416, 928, False, True, False, "train"),
    ("bf16", 33, 1024, 3504, True, False, True, "train"),
    ("bf16", 1, 304, 10360, False, False, True, "train"),                 # 64 columns, whole
    ("bf16", 17, 448, 7112, False, True, False, "train"),
    ("bf16", 33, 512, 6184, False, False, True, "train"),
    ("bf16", 4178, 2200, 200, True, True, True, "train"),
    ("bf16", 1194, 1000, 1672, False, True, False, "train"),
    ("bf16", 2553, 1008, 800, True, False, True, "train"),
    ("bf16", 334, 1992, 3544, False, True, True, "train"),
    ("bf16", 453, 2032, 2624, True, False, False, "train"),
    ("bf16", 3626, 1008, 1056, True, False, True, "train"),
    ("bf16", 264, 4112, 3736, False, False, False, "train"),
    ("bf16", 2488, 856, 2528, False, False, True, "train"),
    ("bf16", 5161, 1216, 1712, False, True, True, "train"),
    ("bf16", 5110, 856, 2472, True, True, False, "train"),
    ("bf16", 4585, 840, 2888, False, False, False, "train"),
    ("bf16", 5352, 3232, 1424, True, True, True, "train"),
    ("bf16", 4809, 2840, 3504, False, True, True, "train"),
    ("bf16", 4825, 2520, 4072, True, False, True, "train"),
    ("bf16", 2712, 4776, 1520, True, False, True, "train"),              # largest tiles, split
    ("bf16", 2715, 4784, 1512, False, True, True, "train"),
    ("bf16", 904, 7056, 1368, True, True, True, "train"),
    ("bf16", 901, 7064, 1352, False, False, False, "train"),
    ("f32", 1, 8, 8, False, False, True, "graph"),
    ("f32", 1, 8, 8, True, False, False, "graph"),
    ("f32", 18, 8, 8, True, True, False, "graph"),
    ("f32", 19, 8, 8, False, True, False, "graph"),
    ("f32", 33, 8, 8, False, False, True, "graph"),
    ("f32", 34, 12, 8, True, True, False, "graph"),
    ("f32", 66, 8, 8, False, True, False, "train"),
    ("f32", 1, 1388, 8, True, True, False, "train"),
    ("f32", 68, 248, 8, False, False, False, "train"),
    ("f32", 25, 1028, 8, False, False, False, "train"),
    ("f32", 46, 1176, 8, True, True, False, "train"),
    ("f32", 21, 1164, 1076, True, False, True, "graph"),
    ("f32", 37, 1048, 540, False, False, True, "train"),
    ("f32", 1, 1744, 1804, False, False, True, "train"),
    ("f32", 18, 1280, 1240, True, True, True, "train"),
    ("f32", 1878, 8, 3268, True, True, True, "train"),
    ("f32", 985, 68, 3112, True, True, True, "train"),
    ("f32", 5479, 372, 144, True, False, True, "train"),
    ("f32", 4489, 100, 684, False, False, True, "train"),
    ("f32", 4733, 388, 204, False, True, True, "train"),
    ("f32", 4156, 952, 132, True, False, True, "train"),
    ("f32", 616, 1368, 1220, False, True, True, "train"),
    ("f32", 2947, 1744, 356, True, False, True, "train"),
    ("f32", 2017, 952, 2240, True, True, True, "train"),
    ("f32", 3957, 976, 1140, False, False, True, "train"),
]

# rows, values: by 8 to 1024 threads a row, of whole chunks and not, more rows than a
# launch has places for
NORM = [(70001, 56), (91, 61), (33001, 120), (87, 127), (33, 200), (8199, 251), (8200, 264), (77, 509),
        (31, 776), (8197, 1021), (2051, 1544), (19, 2047), (2050, 2504), (23, 4095), (2053, 5000),
        (11, 8191), (13, 9000), (517, 16381)]


@pytest.fixture(autouse=True)
def references_on_the_gpu(monkeypatch):
    monkeypatch.setattr(dense, "wide", lambda t: None if t is None else t.detach().double())


def kernels_that_run(call):
    """(the call's results, the dense operators' kernels it launched)"""
    call()
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as prof:
        out = call()
        torch.cuda.synchronize()
    names = {V.plain_name(e.key) for e in prof.key_averages()}
    return out, names - {None}


def run(forward, leaves, gy, how):
    """Output and gradients of the named leaves, held to the bits of a call that records
    nothing, and the kernels that ran (graph: outside of it, within it)."""
    if how == "train":
        def call():
            y = forward()
            return [y, *torch.autograd.grad(y, list(leaves.values()), gy)]
        got, ran = kernels_that_run(call)
        with torch.no_grad():
            assert torch.equal(forward(), got[0])
        return dict(zip(("y", *leaves), got)), [ran]
    with torch.no_grad():
        y, eager = kernels_that_run(forward)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = forward()
        out.fill_(1)
        _, ran = kernels_that_run(lambda: [graph.replay() for _ in range(3)])
        assert torch.equal(out, y)
    return {"y": y}, [eager, ran]


def hold_kernels(ran, of, how):
    """The kernels that ran are those that _dense_variants.py says. (The profiler at
    times sees none of a graph's.)"""
    if how == "train":
        assert ran == [set(of(train=True))]
    else:
        eager, captured = (set(of(train=False, captured=c)) for c in (False, True))
        assert ran[0] == eager and (not ran[1] or ran[1] == captured), ran


@pytest.mark.parametrize("case", LINEAR, ids=lambda c: "-".join(map(str, c[:5])))
def test_fused_linear(case, device):
    dt, rows, k, n, transposed, act, bias, residual, how = case
    t = DTYPE[dt]
    g = gen(rows + 7 * k + 11 * n)
    x, w = rnd(g, rows, k, dtype=t), matrix(g, k, n, t, transposed)
    b = rnd(g, n, dtype=t, std=0.5) if bias else None
    r = rnd(g, rows, n, dtype=t) if residual else None
    gy = rnd(g, rows, n, dtype=t)
    leaves = {i: v.requires_grad_() for i, v in (("x", x), ("w", w), ("b", b), ("r", r)) if v is not None}
    got, ran = run(lambda: K.fused_linear(x, w, b, act, r), leaves, gy, how)
    hold_kernels(ran, partial(V.linear, dt, rows, k, n, transposed, act, bias, residual), how)
    ref, tol = linear_reference(x, w, b, r, gy, act)
    for name, v, q in zip(("y", "x", "w", "b"), ref, tol):
        if name in got:
            o = got[name]
            close(o, v, q + half(o) * (v.abs() + q), name, 1 if name in "yb" else 2)
    if "r" in got:
        assert torch.equal(got["r"], gy)


@pytest.mark.parametrize("case", GATED, ids=lambda c: "-".join(map(str, c[:6])))
def test_gated_mlp(case, device):
    dt, rows, d, width, t1, t2, bias, how = case
    t = DTYPE[dt]
    act = sorted(GATES)[(rows + d // 4 + width // 4) % 4]
    g = gen(rows + 7 * d + 11 * width)
    x = rnd(g, rows, d, dtype=t)
    w1, w2 = matrix(g, d, 2 * width, t, t1), matrix(g, width, d, t, t2)
    b1 = rnd(g, 2 * width, dtype=t, std=0.5) if bias else None
    b2 = rnd(g, d, dtype=F32, std=0.5) if bias else None
    r = rnd(g, rows, d, dtype=t) if t1 else None
    gy = rnd(g, rows, d, dtype=t)
    leaves = {i: v.requires_grad_() for i, v in (("x", x), ("w1", w1), ("w2", w2), ("b1", b1), ("b2", b2),
                                                 ("r", r)) if v is not None}
    got, ran = run(lambda: K.gated_mlp(x, w1, w2, act, b1, b2, r), leaves, gy, how)
    hold_kernels(ran, partial(V.gated, dt, rows, d, width, t1, t2, bias), how)
    ref, tol = gated_reference(x, w1, w2, b1, b2, r, gy, act)
    for name, v, q in zip(("y", "x", "w1", "w2", "b1", "b2"), ref, tol):
        if name in got:
            o = got[name]
            close(o, v, q + half(o) * (v.abs() + q), f"{act} {name}", 2)
    if "r" in got:
        assert torch.equal(got["r"], gy)


@pytest.mark.parametrize("dtype", list(DTYPE))
@pytest.mark.parametrize("rows,d", NORM)
def test_layer_norm(rows, d, dtype, device):
    t = DTYPE[dtype]
    g = gen(rows + d)
    x, gy = rnd(g, rows, d, dtype=t, mean=0.5).requires_grad_(), rnd(g, rows, d, dtype=t)
    w, b = rnd(g, d, mean=1.0, std=0.2), rnd(g, d, dtype=t, std=0.2)
    for weights in (False, True):
        leaves = {"x": x, "w": w.requires_grad_(), "b": b.requires_grad_()} if weights else {"x": x}
        args = (x, w, b) if weights else (x,)
        got, ran = run(lambda: K.layer_norm(*args), leaves, gy, "train")
        assert ran == [set(V.norm(dtype, rows, d, True, weights))]
        one = (w, b) if weights else (torch.ones_like(w), torch.zeros_like(w))
        ref, tol = norm_reference(x, *one, gy, 1e-5)
        for name, v, q in zip(("y", "x", "w", "b"), ref, tol):
            if name in got:
                close(got[name], v, q + half(got[name]) * v.abs(), name)

"""Every kernel that the few-token operators can take, against the plain 64-bit
implementations of test_gpu_few_tokens.py and with its bounds; and the launch
rules of _few_variants.py, against the kernels that run."""

from __future__ import annotations

import pytest
import torch
from torch.profiler import ProfilerActivity, profile

import _few_variants as V
import test_gpu_few_tokens as few
from test_gpu_few_tokens import D, U16, U32, expand, hold, layer_inputs, normal, plain_experts, \
    plain_quantized
from triton_moe import kernels as K

pytestmark = pytest.mark.gpu

GLU, RELU = "swiglu", "relu_squared"
CASES = [
    # d, experts, k, T, dtype, group, act: what the other lists do not reach
    (200, "18x72,2x136", 3, 5, "bf16", 0, GLU),   # fewer pairs than experts, by experts
    (200, "300x8", 3, 9, "bf16", 0, GLU),         # the same, whole tiles
    (72, "20x1032", 3, 65, "bf16", 0, GLU),       # whole tiles, two row tiles
    (1032, "20x1032", 3, 5, "bf16", 0, RELU),     # down: weights after the rows, long K
    (2056, "258x8", 2, 65, "bf16", 0, RELU),      # the same, short K
    (200, "18x72,2x136", 3, 5, "f32", 0, RELU),
    (200, "18x72,2x136", 3, 5, "f32", 0, GLU),
    (136, "3x68,2x20", 3, 3, "f32", 0, GLU),
    (200, "300x8", 3, 9, "f32", 0, RELU),
    (200, "300x8", 3, 9, "f32", 0, GLU),
    (72, "20x1032", 4, 5, "f32", 0, GLU),
    (72, "20x1032", 3, 65, "f32", 0, RELU),
    (72, "20x1032", 3, 65, "f32", 0, GLU),
    (2056, "130x8", 2, 33, "f32", 0, RELU),
    (264, "32x136", 4, 4, "q4", 64, RELU),        # a pair a workgroup, narrow tiles
    (264, "32x136", 4, 4, "q4", 128, RELU),
    (264, "32x136", 4, 4, "q4", 32, GLU),
    (264, "32x136", 4, 4, "q4", 128, GLU),
    (648, "18x72,2x136", 3, 5, "q4", 32, RELU),   # fewer pairs than experts, by experts
    (264, "18x72,2x136", 3, 5, "q4", 64, RELU),
    (648, "18x72,2x136", 3, 5, "q4", 128, RELU),
    (648, "18x72,2x136", 3, 5, "q4", 64, GLU),
    (264, "18x72,2x136", 3, 5, "q4", 128, GLU),
    (264, "3x136,2x72", 3, 9, "q4", 64, GLU),
    (520, "300x8", 3, 9, "q4", 32, RELU),         # whole tiles
    (520, "300x8", 3, 9, "q4", 64, RELU),
    (520, "130x72", 2, 65, "q4", 64, RELU),
    (520, "130x72", 2, 65, "q4", 128, RELU),
    (2056, "3x72", 1, 65, "q4", 32, RELU),        # down: one wave along K
    (2056, "3x72", 1, 65, "q4", 128, RELU),
    (1984, "8x1288", 1, 7, "q4", 32, RELU),       # down: fewer pairs than experts
    (1984, "8x1288", 1, 7, "q4", 64, RELU),
    (1984, "8x1288", 1, 7, "q4", 128, RELU),
    (2056, "130x8", 2, 65, "q4", 32, RELU),       # down: many workgroups
    (2056, "130x8", 2, 65, "q4", 64, RELU),
    (2056, "130x8", 8, 17, "q4", 128, RELU),
    (2056, "8x520", 8, 2, "q4", 64, RELU),
]

PRODUCTS = [
    # K, lengths, T, k (0: no ids), group
    (200, [72, 40, 8, 136, 24], 2, 2, 32),        # fewer pairs than matrices
    (200, [72, 40, 8, 136, 24], 2, 2, 64),
    (200, [72, 40, 8, 136, 24], 2, 2, 128),
    (200, [72], 37, 0, 64),
    (520, [16392], 17, 0, 32),                    # two row tiles, many workgroups
    (520, [16392], 17, 0, 64),
    (520, [16392], 17, 0, 128),
]


def kernels_that_run(call):
    """(call's result, the few-token kernels it launched)."""
    call()  # (tables, workspace sizes)
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as prof:
        out = call()
        torch.cuda.synchronize()
    names = {V.plain_name(e.key) for e in prof.key_averages()}
    return out, {n for n in names if n}


def some_ids(T, k, E, seed):
    """Few different experts, the first and the last among them, and no expert."""
    g = torch.Generator().manual_seed(seed)
    few_of = torch.tensor(sorted({0, E // 2, E - 1}))
    ids = few_of[torch.randint(0, len(few_of), (T, k), generator=g)]
    ids[0, 0], ids[T - 1, k - 1] = E - 1, 0
    if T > 2:
        ids[T // 2, 0] = -1
    return ids


@pytest.mark.parametrize("i", range(len(CASES)))
def test_kernel(device, i):
    d, spec, k, T, dt, group, act = CASES[i]
    widths = expand(spec)
    dtype = torch.float32 if dt == "f32" else torch.bfloat16
    x, _, w1, w2 = layer_inputs(9000 + 10 * i, d, widths, T, act, dtype)
    ids = some_ids(T, k, len(widths), i)
    wts = normal(9005 + 10 * i, T, k, dtype=torch.float32)
    if dt == "q4":
        e = K.quantize_experts(w1.to(device), w2.to(device), widths, act, group)
    else:
        e = K.few_token_experts(w1.to(device), w2.to(device), widths, act)
    a, b, c = x.to(device), ids.to(device), wts.to(device)
    out, ran = kernels_that_run(lambda: K.experts_few_tokens(a, b, c, e))
    assert ran == V.layer_kernels(dt, group, d, widths, k, T, act, router=False)
    # the reference holds the experts that are named
    used = sorted({int(v) for v in ids.unique() if v >= 0})
    glu = 2 if act == GLU else 1
    start = [sum(widths[:n]) for n in used]
    p1 = torch.cat([w1[:, glu * o:glu * (o + widths[n])] for n, o in zip(used, start)], 1)
    p2 = torch.cat([w2[o:o + widths[n]] for n, o in zip(used, start)], 0)
    wide = [widths[n] for n in used]
    if dt == "q4":
        p1 = plain_quantized(p1, [w for w in wide for _ in range(glu)], False, group)[0]
        p2 = plain_quantized(p2, wide, True, group)[0]
    local = torch.full_like(ids, -1)
    for j, n in enumerate(used):
        local[ids == n] = j
    ref, err = plain_experts(x.to(D), local, wts.to(D), p1.to(D), p2.to(D), wide, act, dt != "f32")
    hold(out, ref, err, CASES[i])
    none = ~(ids >= 0).any(dim=1)
    assert (out.cpu()[none] == 0).all()


@pytest.mark.parametrize("rows,lengths,T,k,group", PRODUCTS)
def test_product(device, rows, lengths, T, k, group):
    w, x = normal(211, rows, sum(lengths), std=0.05), normal(212, T, rows)
    q = K.quantize_matrices(w.to(device), lengths, "columns", group)
    v = plain_quantized(w, lengths, False, group)[0]
    a = x.to(device)
    ids = some_ids(T, k, len(lengths), 213) if k else None
    b = None if ids is None else ids.to(device)
    y, ran = kernels_that_run(lambda: K.matvec_q4(a, q, b))
    assert ran == V.matvec_kernels(group, rows, lengths, k, T)
    if not k:
        ref, mag = x.to(D) @ v, x.to(D).abs() @ v.abs()
    else:
        ref, mag = (torch.zeros(T, k, max(lengths), dtype=D) for _ in range(2))
        for t in range(T):
            for s in range(k):
                m = int(ids[t, s])
                o, n = sum(lengths[:m]), lengths[m]
                ref[t, s, :n] = x[t].to(D) @ v[:, o:o + n]
                mag[t, s, :n] = x[t].to(D).abs() @ v[:, o:o + n].abs()
        assert (y.cpu().to(D)[mag == 0] == 0).all()
    hold(y, ref, U16 * ref.abs() + (rows + 8) * U32 * mag)


def test_rules_of_the_other_lists(device):
    """The launch rules over the cases of test_gpu_few_tokens.py."""
    for i, (d, spec, k, T, dt, group, _) in enumerate(few.LAYERS):
        widths, dtype = expand(spec), torch.float32 if dt == "f32" else torch.bfloat16
        x, wr, w1, w2 = (t.to(device) for t in layer_inputs(i, d, widths, T, dtype=dtype))
        e = K.quantize_experts(w1, w2, widths, group_size=group) if dt == "q4" else \
            K.few_token_experts(w1, w2, widths)
        _, ran = kernels_that_run(lambda: K.moe_few_tokens(x, wr, e, k))
        assert ran == V.layer_kernels(dt, group, d, widths, k, T), few.LAYERS[i]

"""The GPU tests' cases reach every kernel that the library holds for the dense
operators, by launch rules that are held to the library's workspace queries here and to
the kernels that run on the GPU."""

from __future__ import annotations

import random
import shutil

import pytest

import _dense_variants as V
import test_gpu_dense_variants as cases
from triton_moe import _lib


def reached():
    parts = []
    for *args, how in cases.LINEAR:
        parts += [V.linear(*args, train=how == "train", captured=c) for c in {False, how == "graph"}]
    for *args, how in cases.GATED:
        parts += [V.gated(*args, train=how == "train", captured=c) for c in {False, how == "graph"}]
    parts += [V.norm(dt, rows, d, True, weights) for dt in V.NAME for rows, d in cases.NORM
              for weights in (False, True)]
    return V.merge(*parts)


@pytest.mark.skipif(shutil.which("nm") is None, reason="needs nm")
def test_every_kernel_is_reached():
    held = V.library_kernels(_lib.LIB_PATH)
    assert len(held) > 200 and set(reached()) == held


def test_every_kind_of_product_is_reached():
    """Tiles: all of them whole, all split along k, and whole ones with a split tail. Few
    rows: whole and split."""
    for kernel, states in reached().items():
        if kernel.startswith(("big_", "gemm_")):
            assert states == {"whole", "split", "both"}, kernel
        elif kernel.startswith("join_kernel"):
            assert states == {"split", "both"}, kernel
        elif kernel.startswith("few_") and ", 3, " not in kernel:
            assert states == {"whole", "split"}, kernel


def test_plans_are_the_library_s():
    """By the workspace of a forward pass: the sums of its split products."""
    lib, r = _lib.lib(), random.Random(3)

    def size(lo, hi, unit=1):
        return max(unit, round(lo * (hi / lo) ** r.random() / unit) * unit)

    split = 0
    for _ in range(4000):
        dt = r.choice(list(V.NAME))
        unit = 16 // V.SIZE[dt]
        rows, k, n = size(1, 40000), size(8, 16384, unit), size(8, 16384, unit)
        code = _lib.DENSE_BF16 if dt == "bf16" else _lib.DENSE_F32

        def sums(epi, *sizes):
            return max(V.plan(dt, form, epi, *sizes).part_bytes for form in (V.KK, V.KT))
        linear, gated = sums(V.LINEAR, rows, n, k), sums(V.GATED, rows, n, k)
        assert lib.vmoe_linear_workspace_bytes(code, rows, k, n, 0, 0) == linear, (dt, rows, k, n)
        assert lib.vmoe_gated_workspace_bytes(code, rows, k, n, 0) == \
            max(gated, sums(V.LINEAR, rows, k, n)), (dt, rows, k, n)
        split += linear > 0
    assert 1000 < split < 4000


def test_names():
    assert V.plain_name("void vmoe::dense::(anonymous namespace)::gemm_kernel<vmoe::dense::Bf16, false, "
                        "true, 1, 64, 128, 2>(vmoe::dense::GemmArgs)") == \
        "gemm_kernel<Bf16, false, true, 1, 64, 128, 2>"
    assert V.plain_name("void vmoe::dense::(anonymous namespace)::act_grad_kernel<vmoe::dense::F32, "
                        "(vmoe::dense::(anonymous namespace)::SlopeOf)1>(void const*, long)") == \
        "act_grad_kernel<F32, 1>"
    assert V.plain_name("vmoe::dense::(anonymous namespace)::col_sum_kernel(float const*)") == \
        "col_sum_kernel"
    assert V.plain_name("void vmoe::route_kernel<1>(int)") is None

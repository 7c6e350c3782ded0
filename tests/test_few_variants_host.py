"""The GPU tests' cases reach every kernel that the library holds for the few-token
operators, by the launch rules that the GPU tests hold to the kernels that run."""

from __future__ import annotations

import shutil

import pytest

import _few_variants as V
import test_gpu_few_tokens as few
import test_gpu_few_variants as more
from triton_moe import _lib


def reached():
    got = set()
    for d, spec, k, T, dt, group, _ in few.LAYERS:
        got |= V.layer_kernels(dt, group, d, few.expand(spec), k, T)
    for d, spec, k, T, dt, group, act, _ in few.EXPERTS:
        got |= V.layer_kernels(dt, group, d, few.expand(spec), k, T, act, router=False)
    for rows, lengths, T, k, group, _ in few.MATVEC:
        got |= V.matvec_kernels(group, rows, lengths, k, T)
    for d, spec, k, T, dt, group, act in more.CASES:
        got |= V.layer_kernels(dt, group, d, few.expand(spec), k, T, act, router=False)
    for rows, lengths, T, k, group in more.PRODUCTS:
        got |= V.matvec_kernels(group, rows, lengths, k, T)
    return got


@pytest.mark.skipif(shutil.which("nm") is None, reason="needs nm")
def test_every_kernel_is_reached():
    held = V.library_kernels(_lib.LIB_PATH)
    assert held and reached() == held


def test_names():
    assert V.plain_name("void vmoe::(anonymous namespace)::few_kernel<vmoe::(anonymous namespace)::"
                        "WQ4<2, 1>, (vmoe::(anonymous namespace)::Mode)0, 1, 2, false, 1, true>"
                        "(vmoe::(anonymous namespace)::FewArgs)") == \
        "few_kernel<WQ4<2, 1>, 0, 1, 2, false, 1, true>"
    assert V.plain_name("vmoe::(anonymous namespace)::few_combine_kernel(int)") == \
        "few_combine_kernel"
    assert V.plain_name("void vmoe::gemm_kernel<1>(int)") is None

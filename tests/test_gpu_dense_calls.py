"""Calls of the dense operators at their edges, on the GPU."""

from __future__ import annotations

import pytest
import torch

from test_dense_calls import WITHOUT_MEMORY, Wrapper, calls, freed
from triton_moe import kernels as K

pytestmark = pytest.mark.gpu


def randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("of", WITHOUT_MEMORY)
def test_operands_without_memory(of, device):
    x, w, v = randn(3, 8), randn(8, 8), randn(8)
    for what, call in calls(x, w, v, of):
        with pytest.raises(NotImplementedError, match=f"{what} has no memory"):
            call()
    for call in (lambda: K.layer_norm(of(x)), lambda: K.fused_linear(of(x), w),
                 lambda: K.gated_mlp(of(x), torch.cat([w, w], 1), w)):
        with pytest.raises(NotImplementedError, match="x has no memory"):
            call()


def test_operands_freed_before_the_backward_pass(device):
    """What the backward pass would read, freed between the passes, and a gradient
    whose values are elsewhere."""
    for i in range(8):
        x, v = randn(3, 8).requires_grad_(), randn(8).requires_grad_()
        w, w1 = randn(8, 8).requires_grad_(), randn(8, 16).requires_grad_()
        y, gone = [(K.layer_norm(x, v), v), (K.layer_norm(x, v), x), (K.fused_linear(x, w), w),
                   (K.fused_linear(x, w), x), (K.gated_mlp(x, w1, w), w1),
                   (K.gated_mlp(x, w1, w), w), (K.gated_mlp(x, w1, w), x),
                   (K.fused_linear(x, w, activation="relu"), None)][i]
        (y if gone is None else gone).detach().untyped_storage().resize_(0)
        with pytest.raises(NotImplementedError, match="no memory"):
            torch.autograd.grad(y, [x, w, w1, v], torch.ones(3, 8, device="cuda"), allow_unused=True)
    x, w = randn(3, 8).requires_grad_(), randn(8, 8)
    for y in (K.layer_norm(x), K.fused_linear(x, w), K.gated_mlp(x, torch.cat([w, w], 1), w)):
        with pytest.raises(NotImplementedError, match="no memory"):
            torch.autograd.grad(y, x, Wrapper(torch.ones(3, 8, device="cuda")))


def test_no_rows_have_no_memory(device):
    x = torch.zeros(0, 8, device="cuda")
    assert freed(x).data_ptr() == 0 and K.layer_norm(x).shape == (0, 8)
    assert K.fused_linear(x, randn(8, 8), residual=x).shape == (0, 8)

"""Calls of the dense operators at their edges, on the GPU."""

from __future__ import annotations

import pytest
import torch

from test_dense_calls import WITHOUT_MEMORY, Wrapper, calls, freed
from triton_moe import _lib
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


def saved(call):
    """(what the call returns, the (shape, type) of each tensor that it saves)"""
    kept = []

    def pack(t):
        kept.append((tuple(t.shape), t.dtype))
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        y = call()
    return y, sorted(kept, key=str)


def subsets(names):
    return [{n for i, n in enumerate(names) if m >> i & 1} for m in range(1, 1 << len(names))]


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("act", [None, "relu", "silu"])
def test_fused_linear_saves_what_it_reads(act, transposed, device):
    """For each set of leaves: nothing is saved that their gradients do not read, and
    they have the bits of the whole pass."""
    bf16, f32 = torch.bfloat16, torch.float32
    full = dict(x=randn(2, 35, 72, seed=1, dtype=bf16), w=randn(72, 40, seed=2, dtype=bf16) * 0.1,
                b=randn(40, seed=3), r=randn(2, 35, 40, seed=4, dtype=bf16))
    if transposed:
        full["w"] = full["w"].t().contiguous().t()
    gy = randn(2, 35, 40, seed=5, dtype=bf16)
    for residual in (False, True):
        names = [n for n in full if residual or n != "r"]

        def run(leaves):
            t = {n: full[n].detach().requires_grad_(n in leaves) for n in names}
            y, kept = saved(lambda: K.fused_linear(t["x"], t["w"], t["b"], act, t.get("r")))
            return kept, dict(zip(sorted(leaves), torch.autograd.grad(y, [t[n] for n in sorted(leaves)], gy)))
        _, whole = run(set(names))
        for leaves in subsets(names):
            kept, grads = run(leaves)
            want = [((2, 35, 72), bf16)] if "w" in leaves else []
            want += [((72, 40), bf16)] if "x" in leaves else []
            if leaves - {"r"} and act:
                want += [((2, 35, 40), bf16)] if act == "relu" and not residual else [((70, 40), f32)]
            assert kept == sorted(want, key=str), (leaves, kept)
            for n, g in grads.items():
                assert torch.equal(g, whole[n]) and g.dtype == full[n].dtype, (leaves, n)
                assert g.stride() == whole[n].stride()


def test_gated_mlp_saves_what_it_reads(device):
    bf16, f32 = torch.bfloat16, torch.float32
    full = dict(x=randn(70, 72, seed=1, dtype=bf16), w1=randn(72, 80, seed=2, dtype=bf16) * 0.1,
                w2=randn(72, 40, seed=3, dtype=bf16).t() * 0.1, b1=randn(80, seed=4), b2=randn(72, seed=5),
                r=randn(70, 72, seed=6, dtype=bf16))
    gy = randn(70, 72, seed=7, dtype=bf16)

    def run(leaves):
        t = {n: full[n].detach().requires_grad_(n in leaves) for n in full}
        y, kept = saved(lambda: K.gated_mlp(t["x"], t["w1"], t["w2"], "geglu", t["b1"], t["b2"], t["r"]))
        return kept, dict(zip(sorted(leaves), torch.autograd.grad(y, [t[n] for n in sorted(leaves)], gy)))
    _, whole = run(set(full))
    for leaves in subsets(list(full)):
        kept, grads = run(leaves)
        inner = leaves & {"x", "w1", "b1"}
        want = [((70, 72), bf16)] if "w1" in leaves else []
        want += [((72, 80), bf16)] if "x" in leaves else []
        want += [((40, 72), bf16), ((70, 80), f32)] if inner else []
        want += [((70, 40), bf16)] if "w2" in leaves else []
        assert kept == sorted(want, key=str), (leaves, kept)
        for n, g in grads.items():
            assert torch.equal(g, whole[n]) and g.dtype == full[n].dtype, (leaves, n)
            assert g.stride() == whole[n].stride()


def test_layer_norm_saves_what_it_reads(device):
    full = dict(x=randn(70, 72, seed=1), w=randn(72, seed=2), b=randn(72, seed=3, dtype=torch.bfloat16))
    gy = randn(70, 72, seed=4)

    def run(leaves):
        t = {n: full[n].detach().requires_grad_(n in leaves) for n in full}
        y, kept = saved(lambda: K.layer_norm(t["x"], t["w"], t["b"]))
        return kept, dict(zip(sorted(leaves), torch.autograd.grad(y, [t[n] for n in sorted(leaves)], gy)))
    _, whole = run(set(full))
    for leaves in subsets(list(full)):
        kept, grads = run(leaves)
        want = [((70, 72), torch.float32), ((70, 2), torch.float32)]
        want += [((72,), torch.float32)] if "x" in leaves else []
        assert kept == sorted(want, key=str), (leaves, kept)
        for n, g in grads.items():
            assert torch.equal(g, whole[n]) and g.dtype == full[n].dtype, (leaves, n)


def test_what_is_not_read_may_change(device):
    """In place, between the passes: biases, the rows where no weight wants a gradient,
    a weight where the rows do not. (A norm always reads its rows.)"""
    x, w, b, r = randn(9, 72), randn(72, 72, seed=1), randn(72, seed=2), randn(9, 72, seed=3)
    w1 = torch.cat([w, w], 1)
    linear = lambda: K.fused_linear(x, w, b, "gelu", r)  # noqa: E731
    gated = lambda: K.gated_mlp(x, w1, w, "swiglu", None, b, r)  # noqa: E731
    norm = lambda: K.layer_norm(x, w[0], b)  # noqa: E731
    for call, leaf, changed in ((linear, x, (b, r)), (linear, w, (w, b, r)), (linear, b, (x, w, b, r)),
                                (linear, r, (x, w, b, r)), (gated, x, (b, r)), (gated, w, (x, b, r)),
                                (gated, b, (x, w, w1, b, r)), (norm, x, (b,)), (norm, b, (w, b))):
        leaf.requires_grad_()
        want, = torch.autograd.grad(call().sum(), leaf)
        y = call().sum()
        with torch.no_grad():
            for t in changed:
                t.add_(1)
        got, = torch.autograd.grad(y, leaf)
        with torch.no_grad():
            for t in changed:
                t.sub_(1)
        leaf.requires_grad_(False)
        assert torch.equal(got, want)


def test_negative_transposed_weight(device):
    """A view that stands for its negative is read in the order of its copy, and its
    gradient comes in that order, whatever the view's."""
    w = randn(40, 72, seed=1)
    n = torch.complex(torch.zeros_like(w), -w).conj().imag.t()  # [72, 40], strides (2, 144)
    x, gy = randn(70, 72).requires_grad_(), randn(70, 40, seed=2)
    assert n.is_neg() and torch.equal(n, w.t())
    got = [torch.autograd.grad(K.fused_linear(x, v, None, "silu"), (x, v), gy)
           for v in (n.detach().requires_grad_(), w.t().detach().requires_grad_())]
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_an_observer_s_error_reaches_the_caller(device):
    """As it does from the package's other operators, forward and backward."""
    class Timer:
        def __init__(self, bad):
            self.bad, self.seen = bad, []

        def begin(self, name):
            self.note("begin", name)

        def end(self, name):
            self.note("end", name)

        def note(self, *what):
            self.seen.append(what)
            if what == self.bad:
                raise KeyError("observer")

    x = randn(4, 64).requires_grad_()
    for bad, direction in ((("begin", "vmoe_layer_norm"), 0), (("end", "vmoe_layer_norm"), 0),
                           (("begin", "vmoe_layer_norm_backward"), 1),
                           (("end", "vmoe_layer_norm_backward"), 1)):
        y = K.layer_norm(x)
        t = Timer(bad)
        _lib.set_launch_timer(t)
        try:
            with pytest.raises(KeyError, match="observer"):
                y.sum().backward() if direction else K.layer_norm(x)
        finally:
            _lib.set_launch_timer(None)
        assert t.seen[-1] == bad
    K.layer_norm(x).sum().backward()

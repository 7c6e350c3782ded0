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


def step(x, p):
    h = K.fused_linear(K.layer_norm(x, p[0], p[1]), p[2], p[3], "gelu", x)
    return K.gated_mlp(h, p[4], p[5], "swiglu", None, p[3], h)


def parameters(dtype=torch.bfloat16, d=264, width=520):
    p = [randn(d, seed=1), randn(d, seed=2), randn(d, d, seed=3, dtype=dtype) * 0.06,
         randn(d, seed=4, dtype=dtype), randn(2 * width, d, seed=5, dtype=dtype).t() * 0.06,
         randn(width, d, seed=6, dtype=dtype) * 0.04]
    return [t.detach().requires_grad_() for t in p]


@pytest.mark.parametrize("rows", [7, 300])
def test_recomputed_and_moved_aside(rows, device):
    """Under torch's checkpoints, and with what is saved kept on the host: the bits of the
    plain step."""
    from torch.utils.checkpoint import checkpoint

    p, x = parameters(), randn(rows, 264, dtype=torch.bfloat16).requires_grad_()
    gy = randn(rows, 264, seed=9, dtype=torch.bfloat16)
    want = [step(x, p), *torch.autograd.grad(step(x, p), [x, *p], gy)]
    for reentrant in (False, True):
        for t in (x, *p):
            t.grad = None
        y = checkpoint(step, x, p, use_reentrant=reentrant)
        y.backward(gy)
        assert all(torch.equal(a, b) for a, b in zip(want, [y, *(t.grad for t in (x, *p))]))
    with torch.autograd.graph.save_on_cpu():
        y = step(x, p)
    got = [y, *torch.autograd.grad(y, [x, *p], gy)]
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    y = step(x, p)  # twice through one graph
    for _ in range(2):
        got = torch.autograd.grad(y, [x, *p], gy, retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(want[1:], got))


@pytest.mark.parametrize("own_stream", [False, True])
def test_calls_of_several_threads(own_stream, device):
    """On one stream and on streams of their own, products of few rows (which share a
    stream's arrival words) among them."""
    import threading

    p = parameters()
    wide = randn(4096, 520, seed=7, dtype=torch.bfloat16) * 0.02
    xs = [randn(rows, 264, seed=rows, dtype=torch.bfloat16) for rows in (1, 5, 40, 300)]
    fs = [randn(rows, 4096, seed=rows, dtype=torch.bfloat16) for rows in (1, 5, 40, 300)]

    def work(i):
        x = xs[i].detach().requires_grad_()
        y = step(x, p)
        return [y.detach(), *torch.autograd.grad(y.float().sum(), [x, *p]), K.fused_linear(fs[i], wide)]
    want = [work(i) for i in range(4)]
    torch.cuda.synchronize()
    got, errors = [[] for _ in xs], []

    def thread(i):
        try:
            s = torch.cuda.Stream() if own_stream else torch.cuda.default_stream()
            with torch.cuda.stream(s):
                for _ in range(20):
                    got[i].append(work(i))
        except BaseException as e:  # noqa: BLE001 - raised below
            errors.append(e)

    threads = [threading.Thread(target=thread, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for w, runs in zip(want, got):
        assert len(runs) == 20
        for r in runs:
            assert all(torch.equal(a, b) for a, b in zip(w, r))


def test_transforms_are_refused(device):
    """A batched or traced tensor's values are not in its own memory."""
    x, w = randn(3, 4, 8), randn(8, 8)
    with pytest.raises(NotImplementedError, match="x has no memory"):
        torch.vmap(lambda t: K.fused_linear(t, w))(x)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.grad(lambda t: K.layer_norm(t).sum())(x)


def test_a_call_among_fake_tensors_leaves_nothing(device):
    """Where torch makes tensors without memory a call fails; what a stream keeps is not
    made of them."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    x, w = randn(2, 4096), randn(4096, 64, seed=1)
    want = K.fused_linear(x, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(Exception):
            K.fused_linear(x, w)
        got = K.fused_linear(x, w)
    torch.cuda.synchronize()
    assert torch.equal(got, want)

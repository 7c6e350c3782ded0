"""The few-token and 4-bit entry points called from compiled programs, on the
host: the library gets addresses, so every tensor behind one has to live until
the launch. The library's calls are replaced by a recorder; nothing is launched."""

from __future__ import annotations

import contextlib
import gc

import pytest
import torch

from triton_moe import kernels as K
from triton_moe.kernels import few_tokens as ft

D, WIDTHS, T, TOP_K = 64, [64, 64, 32], 5, 2

# where a library call's arguments hold addresses of tensors (and not None)
ADDRESSES = {
    "vmoe_few_layer": {"x": 1, "router": 4, "out": 8, "selected": 10, "weights": 11, "workspace": 12},
    "vmoe_few_experts": {"x": 1, "ids": 4, "weights": 6, "out": 9, "workspace": 11},
    "vmoe_q4_matvec": {"x": 0, "ids": 3, "codes": 6, "scales": 7, "table": 8, "y": 13},
    "vmoe_q4_quantize": {"w": 0, "table": 3, "codes": 9, "scales": 10},
    "vmoe_q4_dequantize": {"codes": 0, "scales": 1, "table": 2, "out": 8},
}


def storages():
    """(start, end) of the memory of every tensor that is alive."""
    spans = set()
    for t in gc.get_objects():
        if type(t) in (torch.Tensor, torch.nn.Parameter) and t.device.type == "cpu":
            s = t.untyped_storage()
            if s.nbytes():
                spans.add((s.data_ptr(), s.data_ptr() + s.nbytes()))
    return spans


@pytest.fixture
def calls(monkeypatch):
    """The library calls made, each as {argument: the live memory it points into
    (None: into none)}."""
    made = []

    @torch.compiler.disable
    def record(name, *args):
        live = storages()
        where = {}
        for what, i in ADDRESSES[name].items():
            if args[i] is not None:
                where[what] = next((s for s in live if s[0] <= args[i] < s[1]), None)
        made.append((name, where))

    monkeypatch.setattr(ft._lib, "require_gpu", lambda *a: None)
    monkeypatch.setattr(ft._lib, "call", record)
    monkeypatch.setattr(ft._lib, "stream", lambda device: 0)
    monkeypatch.setattr(ft, "_on", lambda device: contextlib.nullcontext())
    torch.compiler.reset()
    yield made
    torch.compiler.reset()


def operands(dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(1)

    def n(*shape):
        return torch.randn(*shape, generator=g).to(dtype)

    return n(T, D), n(len(WIDTHS), D), n(D, sum(WIDTHS)), n(sum(WIDTHS), D)


def strided(t):
    """The same values, columns first in memory: the operators copy such rows."""
    return t.t().contiguous().t()


def entry_points():
    x, wr, w1, w2 = operands()
    ids = torch.randint(0, len(WIDTHS), (T, TOP_K), generator=torch.Generator().manual_seed(2))
    wts = torch.rand(T, TOP_K)
    e = K.few_token_experts(w1, w2, WIDTHS)
    q = K.quantize_experts(w1, w2, WIDTHS)
    return {
        "layer": (lambda x: K.moe_few_tokens(x, strided(wr), e, TOP_K), x),
        "layer_routing": (lambda x: K.moe_few_tokens(x, strided(wr), e, TOP_K, True, True), x),
        "layer_q4": (lambda x: K.moe_few_tokens(x, strided(wr), q, TOP_K), x),
        "experts": (lambda x: K.experts_few_tokens(x, strided(ids), strided(wts), e), x),
        "matvec": (lambda x: K.matvec_q4(x, q.w1, strided(ids)), x),
        "quantize_matrices": (lambda w: K.quantize_matrices(w, WIDTHS).codes, w1),
        "quantize_experts": (lambda w: K.quantize_experts(w, w2, WIDTHS).w2.codes, w1),
        "handle": (lambda w: K.moe_few_tokens(x, strided(wr), K.few_token_experts(w, w2, WIDTHS),
                                              TOP_K), w1),
        "class": (lambda w: K.QuantizedMatrices(w, WIDTHS, "columns", 32).codes, w1),
        "dequantize": (lambda w: q.dequantize()[0] + w, w1),
    }


@pytest.mark.parametrize("name", ["layer", "layer_routing", "layer_q4", "experts", "matvec",
                                  "quantize_matrices", "quantize_experts", "handle",
                                  "class", "dequantize"])
def test_addresses_are_alive_at_the_launch(calls, name):
    call, x = entry_points()[name]
    x = strided(x) if name in ("layer", "layer_routing", "layer_q4", "experts", "matvec") else x
    del calls[:]
    want = call(x)
    eager = [c for c in calls]
    assert eager and all(s for _, where in eager for s in where.values())
    compiled = torch.compile(lambda v: call(v + 0) if x.stride(-1) == 1 else call(strided(v + 0)),
                             backend="eager")
    for _ in range(2):  # (the first call traces, the second runs what was compiled)
        del calls[:]
        got = compiled(x)
        assert got is not None and type(got) is type(want)
        assert [n for n, _ in calls] == [n for n, _ in eager]
        for fn, where in calls:
            assert where.keys() == dict(eager)[fn].keys()
            dead = [what for what, s in where.items() if s is None]
            assert not dead, (fn, dead)
            # what is written shares no memory with what is read, or with other outputs
            written = [w for w in ("out", "workspace", "selected", "weights", "y")
                       if w in where and (fn, w) != ("vmoe_few_experts", "weights")]
            for w in written:
                assert all(where[o] != where[w] for o in where if o != w), (fn, w)


def test_operators_compiled_directly(calls):
    """torch.compile(operator) itself, as opposed to a program that calls it."""
    x, wr, w1, w2 = operands()
    e = K.few_token_experts(w1, w2, WIDTHS)
    layer = torch.compile(K.moe_few_tokens, backend="eager")
    for _ in range(2):
        del calls[:]
        out = layer(strided(x), strided(wr), e, TOP_K)
        assert out.shape == (T, D) and len(calls) == 1
        assert all(calls[0][1].values()), calls


def test_operators_keep_their_documentation():
    for f in (K.moe_few_tokens, K.experts_few_tokens, K.matvec_q4, K.quantize_matrices,
              K.quantize_experts, K.few_token_experts):
        assert f.__doc__ and f.__name__ in K.__all__

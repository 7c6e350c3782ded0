"""Refusals and queries of the few-token and 4-bit entry points, on the host: no
call here reaches a launch."""

from __future__ import annotations

import ctypes

import pytest
import torch

from triton_moe import _lib
from triton_moe import kernels as K
from triton_moe.kernels.few_tokens import _FewWeights

P = 0x1000  # an aligned address that nothing here reads


def weights(**kw):
    w = dict(format=_lib.FEW_BF16, group=0, act=_lib.ACT_RELU_SQUARED, num_experts=4, hidden=64,
             max_width=64, w1=P, scales1=None, ldw1=256, table1=P, w2=P, scales2=None, ldw2=64,
             table2=P, tiles1=P, num_tiles1=4)
    w.update(kw)
    return _FewWeights(*(w[f] for f, _ in _FewWeights._fields_))


def layer(w, T=1, k=2, x=P, ldx=64, wr=P, ldwr=64, out=P, ldo=64, ws=P, n=1 << 30):
    return _lib.lib().vmoe_few_layer(ctypes.addressof(w), x, ldx, T, wr, ldwr, k, 1, out, ldo,
                                     None, None, ws, n, None)


def experts(w, T=1, k=2, ids=P, wts=P, x=P, ldx=64, out=P, ldo=64, ws=P, n=1 << 30):
    return _lib.lib().vmoe_few_experts(ctypes.addressof(w), x, ldx, T, ids, 0, wts, 0, k, out,
                                       ldo, ws, n, None)


BAD = _lib.ERR_INVALID_ARG
NOT = _lib.ERR_UNSUPPORTED


@pytest.mark.parametrize("change,status", [
    (dict(format=3), BAD), (dict(format=-1), BAD), (dict(act=_lib.ACT_NONE), BAD),
    (dict(num_experts=0), BAD), (dict(hidden=0), BAD), (dict(max_width=-8), BAD),
    (dict(w1=None), BAD), (dict(w2=None), BAD), (dict(table1=None), BAD), (dict(table2=None), BAD),
    (dict(tiles1=None), BAD), (dict(num_tiles1=0), BAD), (dict(ldw1=0), BAD), (dict(ldw2=56), BAD),
    (dict(hidden=68, ldw2=72), NOT), (dict(max_width=60), NOT), (dict(ldw1=260), NOT),
    (dict(w1=P + 8), NOT), (dict(table2=P + 4), NOT), (dict(num_experts=2049), NOT),
    (dict(ldw1=(1 << 24) + 8), NOT), (dict(hidden=(1 << 24) + 8, ldw2=(1 << 24) + 8), NOT),
    (dict(format=_lib.FEW_Q4, group=32), BAD),  # no scales
    (dict(format=_lib.FEW_Q4, group=16, scales1=P, scales2=P), BAD),
    (dict(format=_lib.FEW_Q4, group=64, scales1=P + 2, scales2=P), NOT),
    (dict(format=_lib.FEW_F32, hidden=66, ldw2=66), NOT),
])
def test_weights_are_checked(change, status):
    assert layer(weights(**change)) == status
    assert experts(weights(**change)) == status


@pytest.mark.parametrize("change,status", [
    (dict(T=-1), BAD), (dict(k=0), BAD), (dict(x=None), BAD), (dict(out=None), BAD),
    (dict(ws=None), BAD), (dict(ldx=56), BAD), (dict(ldo=56), BAD),
    (dict(T=257), NOT), (dict(k=65), NOT), (dict(ldx=68), NOT), (dict(x=P + 2), NOT),
    (dict(out=P + 8), NOT), (dict(ws=P + 4), NOT), (dict(T=256, ldx=1 << 27), NOT),
    (dict(n=255), _lib.ERR_WORKSPACE),
])
def test_calls_are_checked(change, status):
    assert layer(weights(num_experts=80), **change) == status
    assert experts(weights(num_experts=80), **change) == status


def test_calls_are_checked_each():
    w = weights()
    assert layer(w, k=5) == BAD  # more experts a token than there are
    assert layer(w, wr=None) == BAD and layer(w, ldwr=56) == BAD
    assert layer(w, wr=P + 2) == NOT
    assert experts(w, ids=None) == BAD and experts(w, wts=None) == BAD
    assert experts(w, T=256, k=17) == NOT  # more than 4096 pairs
    assert layer(w, T=0, x=None, out=None, ws=None) == _lib.OK
    assert experts(w, T=0, x=None, out=None, ids=None) == _lib.OK
    assert _lib.lib().vmoe_few_layer(None, P, 64, 1, P, 64, 2, 1, P, 64, None, None, P, 1 << 20,
                                     None) == BAD
    # activations of 4 GiB and more
    big = weights(max_width=1 << 20, ldw1=1 << 20)
    assert experts(big, T=256, k=4, n=1 << 62) == NOT


def test_workspace_query():
    L = _lib.lib()
    n = L.vmoe_few_workspace_bytes(64, 64, 8, 1024, 256, _lib.FEW_BF16)
    # logits, the choice, h in two halves, y
    assert n >= 64 * 64 * 4 + 512 * (8 + 16 + 256 * 4 + 1024 * 4)
    assert L.vmoe_few_workspace_bytes(0, 64, 8, 1024, 256, _lib.FEW_BF16) > 0
    for bad in ((-1, 64, 8, 1024, 256, 0), (1, 0, 8, 1024, 256, 0), (1, 64, 0, 1024, 256, 0),
                (1, 64, 8, 0, 256, 0), (1, 64, 8, 1024, 0, 0), (1, 64, 8, 1024, 256, 3)):
        assert L.vmoe_few_workspace_bytes(*bad) == 0
    assert L.vmoe_few_max_tokens() == K.few_tokens_max() == 256


def matvec(x=P, ldx=64, T=1, ids=P, k=1, codes=P, scales=P, table=P, M=2, rows=64, cols=64,
           group=32, y=P, ldy=64):
    return _lib.lib().vmoe_q4_matvec(x, ldx, T, ids, 0, k, codes, scales, table, M, rows, cols,
                                     group, y, ldy, None)


@pytest.mark.parametrize("change,status", [
    (dict(x=None), BAD), (dict(y=None), BAD), (dict(codes=None), BAD), (dict(scales=None), BAD),
    (dict(table=None), BAD), (dict(ids=None), BAD), (dict(ids=None, M=1, k=2), BAD),
    (dict(M=0), BAD), (dict(T=-1), BAD), (dict(k=0), BAD), (dict(rows=0), BAD),
    (dict(cols=0), BAD), (dict(group=96), BAD), (dict(ldx=56), BAD), (dict(ldy=56), BAD),
    (dict(rows=60), NOT), (dict(cols=60), NOT), (dict(T=257), NOT), (dict(T=256, k=17), NOT),
    (dict(M=2049), NOT), (dict(codes=P + 8), NOT), (dict(x=P + 2), NOT), (dict(ldy=68), NOT),
    (dict(T=0), _lib.OK),
])
def test_matvec_is_checked(change, status):
    assert matvec(**change) == status


@pytest.mark.parametrize("change,status", [
    (dict(w=None), BAD), (dict(table=None), BAD), (dict(codes=None), BAD), (dict(scales=None), BAD),
    (dict(M=0), BAD), (dict(by_rows=2), BAD), (dict(fixed=0), BAD), (dict(max_len=0), BAD),
    (dict(group=0), BAD), (dict(ld=0), BAD), (dict(ld=56), BAD), (dict(by_rows=1, ld=120), BAD),
    (dict(M=65536), NOT), (dict(codes=P + 4), NOT), (dict(fixed=(1 << 28) + 8), NOT),
])
def test_quantize_is_checked(change, status):
    a = dict(w=P, ld=128, table=P, M=2, by_rows=0, fixed=128, max_len=64, group=32, codes=P,
             scales=P)
    a.update(change)
    L = _lib.lib()
    assert L.vmoe_q4_quantize(a["w"], 0, a["ld"], a["table"], a["M"], a["by_rows"], a["fixed"],
                              a["max_len"], a["group"], a["codes"], a["scales"], None) == status
    assert L.vmoe_q4_dequantize(a["codes"], a["scales"], a["table"], a["M"], a["by_rows"],
                                a["fixed"], a["max_len"], a["group"], a["w"], 0, a["ld"],
                                None) == status


def test_host_tensors_are_refused():
    """No CPU fallback, as everywhere in the package."""
    w1, w2 = torch.zeros(64, 128), torch.zeros(128, 64)
    with pytest.raises(AssertionError, match="CUDA"):
        K.few_token_experts(w1, w2, [64, 64])
    with pytest.raises(AssertionError, match="CUDA"):
        K.quantize_experts(w1, w2, [64, 64])
    with pytest.raises(AssertionError, match="CUDA"):
        K.quantize_matrices(w1)
    for widths in ([], [64, 0], [-64, 128]):
        with pytest.raises(ValueError, match="widths"):
            K.quantize_experts(w1, w2, widths)
    with pytest.raises(ValueError, match="group_size"):
        K.quantize_matrices(w1, group_size=48)
    with pytest.raises(ValueError, match="stacked"):
        K.quantize_matrices(w1, stacked="diagonal")


@pytest.fixture
def host_handles(monkeypatch):
    """Handles made of host tensors with nothing launched; the library calls
    that operators make of them afterwards."""
    from triton_moe.kernels import few_tokens as ft

    made = []
    with monkeypatch.context() as m:
        m.setattr(ft._lib, "require_gpu", lambda *a: None)
        m.setattr(ft._lib, "call", lambda *a: None)
        m.setattr(ft._lib, "stream", lambda d: 0)
        m.setattr(ft, "_on", lambda d: __import__("contextlib").nullcontext())
        w1 = torch.randn(64, 128).to(torch.bfloat16)
        w2 = torch.randn(128, 64).to(torch.bfloat16)
        few, four = K.few_token_experts(w1, w2, [64, 64]), K.quantize_experts(w1, w2, [64, 64])
    monkeypatch.setattr(ft._lib, "call", lambda *a: made.append(a))
    monkeypatch.setattr(ft._lib, "stream", lambda d: 0)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    return few, four, made


@pytest.mark.parametrize("saved_from", ["cuda:0", "cuda:1"])
def test_a_loaded_handle_is_where_its_tensors_are(host_handles, saved_from):
    """A handle saved on a GPU and loaded elsewhere (torch.load with a
    map_location) must not hand over addresses of another device: it is used where
    its tensors are, and on the host not at all."""
    import pickle

    few, four, made = host_handles
    for h in (few, four, four.w1, four.w2):
        h.device = torch.device(saved_from)
    few, four = pickle.loads(pickle.dumps((few, four)))
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    wr = torch.zeros(2, 64, dtype=torch.bfloat16)
    ids = torch.zeros(2, 1, dtype=torch.int64)
    for h in (few, four, four.w1, four.w2):
        assert h.device == torch.device("cpu")
    for call in (lambda: K.moe_few_tokens(x, wr, few, 1), lambda: K.moe_few_tokens(x, wr, four, 1),
                 lambda: K.experts_few_tokens(x, ids, torch.ones(2, 1), few),
                 lambda: K.experts_few_tokens(x, ids, torch.ones(2, 1), four),
                 lambda: K.matvec_q4(x, four.w1, ids), lambda: four.dequantize()):
        with pytest.raises(AssertionError, match="CUDA"):
            call()
    assert not made

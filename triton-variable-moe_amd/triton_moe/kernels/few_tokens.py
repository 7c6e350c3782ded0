"""The expert layer for a few tokens (a generation step), in bf16, fp32 or with
4-bit expert weights, and products of rows with 4-bit matrices
(csrc/few_tokens.hip, csrc/few_q4.hip). Inference only: nothing here records
gradients. The reference has no counterpart; its layer pads each expert's rows
to a block (triton_moe/moe.py:148-250).

A program keeps a handle of its weights, made once:

    experts = few_token_experts(w1, w2, widths)             # the weights themselves
    experts = quantize_experts(w1, w2, widths)              # a 4-bit copy
    out = moe_few_tokens(x, router_weight, experts, top_k)  # the whole layer
    out = experts_few_tokens(x, selected, weights, experts)  # with a router of one's own

and, for a single matrix or a stack of them,

    q = quantize_matrices(w)
    y = matvec_q4(x, q)                                     # x @ w, w in 4 bits

Calls take 1 to few_tokens_max() tokens, run on the current stream of x's
device without a host sync, allocate their output and workspace from torch's
allocator, and can be captured into a graph.

A 4-bit value is 0, 0.5, 1, 1.5, 2, 3, 4 or 6 with a sign, times a bf16 scale
that a group of 32, 64 or 128 values of a column shares along the summed axis.
"""

from __future__ import annotations

import contextlib
import ctypes
import functools
import weakref

import torch

from .. import _lib

_ACT = {"relu_squared": _lib.ACT_RELU_SQUARED, "swiglu": _lib.ACT_SWIGLU}
_GROUPS = (32, 64, 128)
_MAX_PAIRS, _MAX_TOP_K, _MAX_EXPERTS = 4096, 64, 2048
_Q4_ROWS, _Q4_COLS, _Q4_BLOCK = 128, 16, 1024
_TILE = 64  # columns of an up projection's workgroup


@functools.lru_cache(maxsize=None)
def few_tokens_max() -> int:
    """The most tokens (rows of x) a call takes."""
    return int(_lib.lib().vmoe_few_max_tokens())


def _widths_of(widths) -> list[int]:
    if isinstance(widths, torch.Tensor):
        widths = widths.tolist()
    widths = list(map(int, widths))
    if not widths or min(widths) <= 0:
        raise ValueError("expert_widths must hold at least one width, all positive")
    return widths


def _weight(w: torch.Tensor, what: str, dtypes, mult: int) -> torch.Tensor:
    """A weight matrix as the kernels read it: on the GPU, rows contiguous,
    aligned and a multiple of 16 bytes apart. Not copied: a handle's weights are
    the caller's."""
    _lib.require_gpu(w, what)
    if w.dim() != 2:
        raise ValueError(f"{what} must have two dimensions (got {w.dim()})")
    if w.dtype not in dtypes:
        raise NotImplementedError(f"{what} must be one of {dtypes} (got {w.dtype})")
    if w.stride(1) != 1 or w.stride(0) % mult or w.data_ptr() % 16:
        raise NotImplementedError(f"{what} must have contiguous 16-byte aligned rows")
    return w


@functools.lru_cache(maxsize=256)
def _entries(lengths: tuple, fixed: int, by_rows: bool, each: int, device) -> tuple:
    """(int32 [matrices, 4] on the device: start, length, first 4-bit block, first
    tile (of _TILE along that axis; the `each` matrices of an expert count
    once); number of 4-bit blocks). A layout's tables, shared by its handles."""
    rows, off, base, tile = [], 0, 0, 0
    for i, n in enumerate(lengths):
        rows.append((off, n, base, tile))
        k, c = (n, fixed) if by_rows else (fixed, n)
        off, base = off + n, base + -(-k // _Q4_ROWS) * -(-c // _Q4_COLS)
        if i % each == each - 1:
            tile += -(-n // _TILE)
    if off >= 2 ** 31 or base >= 2 ** 31:
        raise NotImplementedError("the matrices are too many or too long")
    return torch.tensor(rows, dtype=torch.int32, device=device), base


@functools.lru_cache(maxsize=256)
def _tiles(widths: tuple, device) -> torch.Tensor:
    """int32 on the device: the expert of each tile of _TILE columns."""
    return torch.tensor([e for e, w in enumerate(widths) for _ in range(-(-w // _TILE))],
                        dtype=torch.int32, device=device)


def _untraced(fn):
    """fn, run as it is also where its caller is compiled: it hands addresses to the
    library, and a traced copy of it may let go of a tensor of which only the address
    is used later (an aligned copy, the workspace) before the launch. (The test is
    0.3 us of a call; torch.compiler.disable alone 0.5.)"""
    plain = torch.compiler.disable(fn)

    @functools.wraps(fn)
    def call(*args, **kwargs):
        if torch.compiler.is_compiling():
            return plain(*args, **kwargs)
        return fn(*args, **kwargs)

    return call


_HERE = contextlib.nullcontext()


def _on(device):
    """The device as the current one (kernels and allocations go to it). (What
    torch.cuda.current_device() reads; a device that holds tensors is initialised.)"""
    if torch._C._cuda_getDevice() == device.index:
        return _HERE
    if device.type != "cuda":
        raise AssertionError(f"weights must be on CUDA (these are on {device})")
    return torch.cuda.device(device)


class _FewWeights(ctypes.Structure):
    """struct vmoe_few_weights."""

    _fields_ = [("format", ctypes.c_int32), ("group", ctypes.c_int32), ("act", ctypes.c_int32),
                ("num_experts", ctypes.c_int32), ("hidden", ctypes.c_int64),
                ("max_width", ctypes.c_int64), ("w1", ctypes.c_void_p),
                ("scales1", ctypes.c_void_p), ("ldw1", ctypes.c_int64),
                ("table1", ctypes.c_void_p), ("w2", ctypes.c_void_p),
                ("scales2", ctypes.c_void_p), ("ldw2", ctypes.c_int64),
                ("table2", ctypes.c_void_p), ("tiles1", ctypes.c_void_p),
                ("num_tiles1", ctypes.c_int32)]


class _Experts:
    """What the two kinds of expert handles share."""

    def _init_common(self, fmt, group, activation, widths, hidden, dtype, device):
        self.expert_widths = widths
        self.num_experts = len(widths)
        self.hidden = hidden
        self.activation = activation
        self.dtype = dtype  # of x and out
        self.device = device
        self._max_width = max(widths)
        self._format = fmt
        self._group = group
        self._tiles = _tiles(tuple(widths), device)
        self._desc = None  # made by the first call, and again after a copy
        self._bytes: dict = {}  # (tokens, top_k) -> workspace bytes

    def __getstate__(self):
        return {**self.__dict__, "_desc": None}

    def __setstate__(self, state):
        # (loaded, perhaps onto another device than it was saved from)
        self.__dict__.update(state)
        self.device = self._tiles.device

    def _new_desc(self, w1, scales1, ld1, table1, w2, scales2, ld2, table2) -> _FewWeights:
        q = _FewWeights(self._format, self._group, _ACT[self.activation], self.num_experts,
                        self.hidden, self._max_width, w1, scales1, ld1, table1, w2, scales2, ld2,
                        table2, self._tiles.data_ptr(), self._tiles.numel())
        q.at = ctypes.addressof(q)
        return q

    def _workspace_bytes(self, T: int, k: int, what: str) -> int:
        """Of a call of this size (refused if it is too large); kept in _bytes."""
        _check_count(T, k, what)
        n = self._bytes[(T, k)] = int(_lib.lib().vmoe_few_workspace_bytes(
            T, self.num_experts, k, self.hidden, self._max_width, self._format))
        return n


def _check_layer(w1, w2, widths, activation):
    if activation not in _ACT:
        raise ValueError(f"Unknown activation: {activation} "
                         f"(expected one of {sorted(_ACT)})")
    glu = 2 if activation == "swiglu" else 1
    d, W = w1.shape[0], sum(widths)
    if w1.shape[1] != glu * W:
        raise ValueError(f"w1 must have {glu * W} columns for these widths (got {w1.shape[1]})")
    if w2.shape != (W, d):
        raise ValueError(f"w2 must be [{W}, {d}] (got {tuple(w2.shape)})")
    if w1.device != w2.device:
        raise ValueError("w1 and w2 must be on one device")
    if w1.dtype != w2.dtype:
        raise ValueError(f"w1 and w2 must have one type (got {w1.dtype} and {w2.dtype})")
    return glu, d


class FewTokenExperts(_Experts):
    """Handle of bf16 or fp32 expert weights: few_token_experts."""

    @torch.compiler.disable
    def __init__(self, w1, w2, expert_widths, activation="relu_squared"):
        f32 = w1.dtype == torch.float32
        mult = 4 if f32 else 8
        types = (torch.bfloat16, torch.float32)
        self.w1, self.w2 = (_weight(w, n, types, mult) for w, n in ((w1, "w1"), (w2, "w2")))
        widths = _widths_of(expert_widths)
        glu, d = _check_layer(w1, w2, widths, activation)
        if d % mult or any(w % mult for w in widths):
            raise NotImplementedError(f"hidden size and widths must be multiples of {mult} "
                                      f"for {w1.dtype} weights")
        self._init_common(_lib.FEW_F32 if f32 else _lib.FEW_BF16, 0, activation, widths, d,
                          w1.dtype, w1.device)
        each = [w for w in widths for _ in range(glu)]
        self._t1, _ = _entries(tuple(each), d, False, glu, w1.device)
        self._t2, _ = _entries(tuple(widths), d, True, 1, w1.device)

    def _weights(self) -> _FewWeights:
        """The description of the weights (the caller holds it during its call);
        where their storage or layout has changed since the last one (module.to,
        .data assigned), it is made anew."""
        a, b = self.w1, self.w2
        q = self._desc
        if (q is None or q.w1 != a.data_ptr() or q.w2 != b.data_ptr() or
                a.dtype is not self.dtype or b.dtype is not self.dtype or
                a.stride() != q.strides[0] or b.stride() != q.strides[1] or
                a.shape != q.shapes[0] or b.shape != q.shapes[1]):
            mult = 4 if self._format == _lib.FEW_F32 else 8
            for w, n in ((a, "w1"), (b, "w2")):
                _weight(w, n, (self.dtype,), mult)
                if w.device != self.device:
                    raise ValueError(f"{n} has moved to {w.device}: make a new handle")
            if _check_layer(a, b, self.expert_widths, self.activation)[1] != self.hidden:
                raise ValueError("w1 and w2 have another hidden size now: make a new handle")
            q = self._new_desc(
                a.data_ptr(), None, a.stride(0), self._t1.data_ptr(), b.data_ptr(), None,
                b.stride(0), self._t2.data_ptr())
            q.strides, q.shapes = (a.stride(), b.stride()), (a.shape, b.shape)
            self._desc = q  # (whole: other threads may use it from here on)
        return q


class ModuleExperts(FewTokenExperts):
    """A layer's handle of its own parameters, which the layer keeps alive and may
    replace: it holds them weakly. Its caller holds them during a call."""

    w1 = property(lambda self: self._w1(), lambda self, w: setattr(self, "_w1", weakref.ref(w)))
    w2 = property(lambda self: self._w2(), lambda self, w: setattr(self, "_w2", weakref.ref(w)))


def few_token_experts(w1, w2, expert_widths, activation="relu_squared") -> FewTokenExperts:
    """Handle of expert weights for moe_few_tokens and experts_few_tokens.

    w1 [hidden, sum(widths)] holds the experts side by side ("swiglu":
    [hidden, 2 sum(widths)], gate and up of an expert next to each other), w2
    [sum(widths), hidden] on top of each other; bf16 or fp32, widths and hidden
    size multiples of 8 (fp32: 4). expert_widths: a list of ints or a tensor
    (read back once). The handle refers to w1 and w2 and sees their updates."""
    return FewTokenExperts(w1, w2, expert_widths, activation)


class QuantizedMatrices:
    """A stack of 4-bit matrices in the kernels' order: quantize_matrices."""

    @torch.compiler.disable
    def __init__(self, w, lengths, stacked: str, group_size: int, each: int = 1):
        if stacked not in ("columns", "rows"):
            raise ValueError(f"stacked must be 'columns' or 'rows' (got {stacked!r})")
        if group_size not in _GROUPS:
            raise ValueError(f"group_size must be one of {_GROUPS} (got {group_size})")
        _weight(w, "w", (torch.bfloat16, torch.float32), 1)
        by_rows = stacked == "rows"
        fixed, total = (w.shape[1], w.shape[0]) if by_rows else (w.shape[0], w.shape[1])
        lengths = [total] if lengths is None else _widths_of(lengths)
        if sum(lengths) != total:
            raise ValueError(f"lengths must add up to the matrix's {total} {stacked}")
        if fixed % 8 or any([n % 8 for n in lengths]):
            raise NotImplementedError("matrix sizes must be multiples of 8")
        if len(lengths) > 65535:
            raise NotImplementedError("at most 65535 matrices")
        self.lengths, self.stacked, self.group_size = lengths, stacked, group_size
        self.fixed, self.total, self.max_len = fixed, total, max(lengths)
        self.device = w.device
        self._sizes: set = set()  # (rows, ids a row) of calls that were checked

        self._table, count = _entries(tuple(lengths), fixed, by_rows, each, w.device)
        with _on(w.device):
            self.codes = torch.empty(count * _Q4_BLOCK, dtype=torch.uint8, device=w.device)
            self.scales = torch.empty(count, _Q4_COLS, _Q4_ROWS // group_size,
                                      dtype=torch.bfloat16, device=w.device)
            _lib.call("vmoe_q4_quantize", w.data_ptr(), int(w.dtype == torch.float32),
                      w.stride(0), self._table.data_ptr(), len(lengths), int(by_rows), fixed,
                      self.max_len, group_size, self.codes.data_ptr(), self.scales.data_ptr(),
                      _lib.stream(w.device))

    def __setstate__(self, state):
        # (loaded, perhaps onto another device than it was saved from)
        self.__dict__.update(state)
        self.device = self.codes.device

    @torch.compiler.disable
    def dequantize(self, dtype=torch.bfloat16) -> torch.Tensor:
        """The values, row-major: float32 exactly, bfloat16 rounded once."""
        if dtype not in (torch.bfloat16, torch.float32):
            raise NotImplementedError(f"dequantize to bfloat16 or float32 (got {dtype})")
        by_rows = self.stacked == "rows"
        shape = (self.total, self.fixed) if by_rows else (self.fixed, self.total)
        with _on(self.device):
            out = torch.empty(shape, dtype=dtype, device=self.device)
            _lib.call("vmoe_q4_dequantize", self.codes.data_ptr(), self.scales.data_ptr(),
                      self._table.data_ptr(), len(self.lengths), int(by_rows), self.fixed,
                      self.max_len, self.group_size, out.data_ptr(), int(dtype == torch.float32),
                      out.stride(0), _lib.stream(self.device))
        return out


def quantize_matrices(w, lengths=None, stacked="columns", group_size=32) -> QuantizedMatrices:
    """A 4-bit copy of w [rows, columns] (bf16 or fp32): one matrix, or several
    of `lengths` columns side by side (stacked="columns") or `lengths` rows on
    top of each other ("rows"), grouped along the rows of each. Sizes are
    multiples of 8; a matrix's last group may be short. The scale is
    bf16(max |w| / 6), values the nearest, ties to the even place; a group that
    holds an infinity or NaN stands for NaN."""
    return QuantizedMatrices(w, lengths, stacked, group_size)


class QuantizedExperts(_Experts):
    """Handle of 4-bit expert weights: quantize_experts."""

    @torch.compiler.disable
    def __init__(self, w1, w2, expert_widths, activation="relu_squared", group_size=32):
        widths = _widths_of(expert_widths)
        for w, n in ((w1, "w1"), (w2, "w2")):
            _weight(w, n, (torch.bfloat16, torch.float32), 1)
        glu, d = _check_layer(w1, w2, widths, activation)
        self.w1 = QuantizedMatrices(w1, [w for w in widths for _ in range(glu)], "columns",
                                    group_size, glu)
        self.w2 = quantize_matrices(w2, widths, "rows", group_size)
        self.group_size = group_size
        self._init_common(_lib.FEW_Q4, group_size, activation, widths, d, torch.bfloat16,
                          w1.device)

    def _weights(self) -> _FewWeights:
        q = self._desc
        if q is None:
            a, b = self.w1, self.w2
            q = self._desc = self._new_desc(
                a.codes.data_ptr(), a.scales.data_ptr(), 0, a._table.data_ptr(),
                b.codes.data_ptr(), b.scales.data_ptr(), 0, b._table.data_ptr())
        return q

    @torch.compiler.disable
    def dequantize(self, dtype=torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
        """(w1, w2) that the 4-bit values stand for, as quantize_experts took them."""
        return self.w1.dequantize(dtype), self.w2.dequantize(dtype)


def quantize_experts(w1, w2, expert_widths, activation="relu_squared",
                     group_size=32) -> QuantizedExperts:
    """A 4-bit copy of expert weights (layout as few_token_experts; bf16 or
    fp32) for moe_few_tokens and experts_few_tokens on bf16 activations. The
    copy does not follow later updates of w1 and w2."""
    return QuantizedExperts(w1, w2, expert_widths, activation, group_size)


def _rows(x: torch.Tensor, width: int, dtype, device, what: str):
    """(x, address, row stride, rows): x as rows of `width` values that the
    kernels can read, copied if they are not contiguous or not 16-byte aligned."""
    if (x.dtype is dtype and x.device == device and x.dim() and x.shape[-1] == width and
            x.is_contiguous()):
        at = x.data_ptr()
        if not at % 16:
            return x, at, width, x.numel() // width
    _lib.require_gpu(x, what)
    if x.dim() < 1 or x.shape[-1] != width:
        raise ValueError(f"{what} must have {width} values in its last dimension "
                         f"(got {tuple(x.shape)})")
    if x.dtype != dtype:
        raise NotImplementedError(f"{what} must be {dtype} with these weights (got {x.dtype})")
    if x.device != device:
        raise ValueError(f"{what} is on {x.device}, the weights on {device}")
    if x.dim() != 2:
        x = x.reshape(-1, width)
    mult = 4 if dtype == torch.float32 else 8
    one = x.shape[0] <= 1  # (the stride of a single row is arbitrary)
    if (x.stride(1) != 1 or x.data_ptr() % 16 or
            (not one and (x.stride(0) % mult or x.stride(0) < width))):
        x = x.clone(memory_format=torch.contiguous_format)
    return x, x.data_ptr(), width if one else x.stride(0), x.shape[0]


def _check_count(T: int, k: int, what: str) -> None:
    if k > _MAX_TOP_K:
        raise NotImplementedError(f"{what} takes at most {_MAX_TOP_K} experts a token (got {k})")
    if T > few_tokens_max() or T * k > _MAX_PAIRS:
        raise NotImplementedError(
            f"{what} takes at most {few_tokens_max()} tokens and {_MAX_PAIRS} token-expert pairs "
            f"(got {T} x {k}); larger batches are the layer's own forward's")


@_untraced
def moe_few_tokens(x, router_weight, experts, top_k: int, normalize: bool = True,
                   return_routing: bool = False):
    """The whole layer for a few tokens: router, top_k experts of each token,
    their weighted sum.

    x [..., hidden] in the handle's type, router_weight [num_experts, hidden] in
    the same type. Logits are fp32 and not rounded; the top_k largest are taken
    (equal ones: the lowest index; NaN above all), with weights sigmoid(logit),
    divided by their sum + 1e-20 if normalize. Returns out like x, and with
    return_routing also the chosen experts int32 [tokens, top_k] (largest logit
    first) and their fp32 weights. (TritonMoEMLP.forward rounds its logits to
    bf16, so that near ties may fall differently there.)"""
    d, E, dev, dtype = experts.hidden, experts.num_experts, experts.device, experts.dtype
    k = int(top_k)
    if not 1 <= k <= E:
        raise ValueError(f"top_k must be between 1 and {E} (got {top_k})")
    if router_weight.dim() != 2 or router_weight.shape[0] != E:
        raise ValueError(f"router_weight must be [{E}, {d}] (got {tuple(router_weight.shape)})")
    rows, at, ldx, T = _rows(x, d, dtype, dev, "x")
    wr, wr_at, ldwr, _ = _rows(router_weight, d, dtype, dev, "router_weight")
    n = experts._bytes.get((T, k)) or experts._workspace_bytes(T, k, "moe_few_tokens")
    q = experts._weights()
    with _on(dev):
        out = torch.empty(x.shape, dtype=dtype, device=dev)
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
        sel = wts = None
        if return_routing:
            sel = torch.empty((T, k), dtype=torch.int32, device=dev)
            wts = torch.empty((T, k), dtype=torch.float32, device=dev)
        _lib.call("vmoe_few_layer", q.at, at, ldx, T, wr_at, ldwr, k,
                  1 if normalize else 0, out.data_ptr(), d, _lib.ptr(sel), _lib.ptr(wts),
                  ws.data_ptr(), n, _lib.stream(dev))
    return (out, sel, wts) if return_routing else out


@_untraced
def experts_few_tokens(x, selected, weights, experts):
    """The experts' part of the layer for given choices: out[t] = sum_s
    weights[t, s] expert_{selected[t, s]}(x[t]).

    x [..., hidden] in the handle's type; selected [..., k] int32 or int64 and
    weights [..., k] bf16 or fp32, a row for each of x. An id outside
    0..num_experts-1 (say -1, for the padding of a batch) is no expert: a token
    without any gets zeros. An expert named twice counts twice."""
    d, dev, dtype = experts.hidden, experts.device, experts.dtype
    rows, at, ldx, T = _rows(x, d, dtype, dev, "x")
    ids, k = _ids(selected, T, dev, "selected")
    if weights.shape != selected.shape:
        raise ValueError(f"weights must have the shape of selected, {tuple(selected.shape)} "
                         f"(got {tuple(weights.shape)})")
    if weights.dtype not in (torch.bfloat16, torch.float32):
        raise NotImplementedError(f"weights must be bfloat16 or float32 (got {weights.dtype})")
    if weights.device != dev:
        raise ValueError(f"weights are on {weights.device}, the experts on {dev}")
    n = experts._bytes.get((T, k)) or experts._workspace_bytes(T, k, "experts_few_tokens")
    q = experts._weights()
    wts = weights if weights.is_contiguous() else weights.contiguous()
    with _on(dev):
        out = torch.empty(x.shape, dtype=dtype, device=dev)
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
        _lib.call("vmoe_few_experts", q.at, at, ldx, T, ids.data_ptr(),
                  int(ids.dtype == torch.int64), wts.data_ptr(),
                  int(wts.dtype == torch.bfloat16), k, out.data_ptr(), d, ws.data_ptr(), n,
                  _lib.stream(dev))
    return out


def _ids(ids, T: int, device, what: str):
    """(contiguous ids, ids a row)."""
    if not ids.is_cuda:
        _lib.require_gpu(ids, what)
    if ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what} must be int32 or int64 (got {ids.dtype})")
    if ids.dim() < 1 or ids.shape[-1] < 1 or ids.numel() != T * ids.shape[-1]:
        raise ValueError(f"{what} must have a row of at least one id for each of {T} rows of x "
                         f"(got {tuple(ids.shape)})")
    if ids.device != device:
        raise ValueError(f"{what} is on {ids.device}, the weights on {device}")
    return (ids if ids.is_contiguous() else ids.contiguous()), ids.shape[-1]


@_untraced
def matvec_q4(x, q: QuantizedMatrices, ids=None):
    """Products of a few rows with 4-bit matrices.

    Without ids, q is one matrix [K, N] and y = x @ q, [..., N] for x [..., K].
    With ids [..., k] (int32 or int64, a row for each of x), q's matrices are
    side by side (stacked="columns") and y[..., s, :] = x @ q_{ids[..., s]},
    [..., k, max N]; columns past a matrix's own and rows whose id names no
    matrix are zeros. bf16, fp32 sums rounded once."""
    if q.stacked != "columns":
        raise NotImplementedError("matvec_q4 takes matrices that are side by side "
                                  "(stacked='columns')")
    K, N, dev = q.fixed, q.max_len, q.device
    rows, at, ldx, T = _rows(x, K, torch.bfloat16, dev, "x")
    if ids is None:
        if len(q.lengths) != 1:
            raise ValueError(f"q holds {len(q.lengths)} matrices: ids must say which")
        k, shape = 1, (*x.shape[:-1], N)
    else:
        if ids.shape[:-1] != x.shape[:-1]:
            raise ValueError(f"ids must have a row for each of x: {tuple(x.shape[:-1])} "
                             f"(got {tuple(ids.shape)})")
        ids, k = _ids(ids, T, dev, "ids")
        shape = (*x.shape[:-1], k, N)
    if len(q.lengths) > _MAX_EXPERTS:
        raise NotImplementedError(f"matvec_q4 takes at most {_MAX_EXPERTS} matrices")
    if (T, k) not in q._sizes:
        _check_count(T, k, "matvec_q4")
        q._sizes.add((T, k))
    with _on(dev):
        y = torch.empty(shape, dtype=torch.bfloat16, device=dev)
        _lib.call("vmoe_q4_matvec", at, ldx, T, _lib.ptr(ids),
                  int(ids is not None and ids.dtype == torch.int64), k, q.codes.data_ptr(),
                  q.scales.data_ptr(), q._table.data_ptr(), len(q.lengths), K, N, q.group_size,
                  y.data_ptr(), N, _lib.stream(dev))
    return y

"""Which kernels a call of the dense operators takes: the launch rules of csrc/dense.hip
and csrc/norm.hip, written down a second time, so that tests can be shown to reach every
kernel the library holds, whole, split and mixed. The host tests hold the plans to the
library's workspace queries, the GPU tests the kernels to those that run."""

from __future__ import annotations

import re
import subprocess
from dataclasses import dataclass

KK, KT, TT = 0, 1, 2            # operands contiguous along k, or (T) along m or n
LINEAR, GATED, GATED_BWD, PARTIAL = 0, 1, 2, 3
CUS = 256
# kernel of tiles -> rows, columns, workgroups a CU, us a stage with 1, 2, 3 of them, us a round
TILES = {"bf16": {256: (256, 256, 1, (1.85,), 14.0), 128: (128, 128, 2, (0.87, 1.15), 4.0),
                  64: (64, 64, 3, (0.45, 0.55, 0.70), 2.0)},
         "f32": {128: (128, 128, 2, (2.03, 3.8), 5.0), 64: (64, 64, 3, (0.68, 1.14, 1.62), 2.0)}}
NAME = {"bf16": "Bf16", "f32": "F32"}
SIZE = {"bf16": 2, "f32": 4}


def up(a, b):
    return -(-a // b)


def align256(n):
    return up(n, 256) * 256


@dataclass
class Plan:
    kernel: object              # 256, 128, 64, or "rows" with `cols` columns
    tiles: int
    whole: int
    splits: int
    part_bytes: int
    cols: int = 0

    @property
    def state(self):
        if self.splits == 1:
            return "whole"
        return "both" if self.whole else "split"


def plan_rows(dt, form, epi, M, N, K):
    if form == TT or epi == GATED_BWD or M > 64:
        return None
    n = 2 * N if epi == GATED else N
    size = n * K * SIZE[dt]
    if M > 16 and size > 32 << 20:
        return None
    cols = 64 if dt == "bf16" and form == KT and size > 12 << 20 else 32
    blocks, stage = up(n, cols), 128 // SIZE[dt]
    most = 1 if K <= 1024 and cols == 32 else up(K, 512)
    s = max(1, min(up(CUS, blocks), most))
    kper = up(up(K, stage), s) * stage
    splits = up(K, kper)
    return Plan("rows", blocks, 0, splits,
                align256(splits * M * blocks * cols * 4) if splits > 1 else 0, cols)


def plan(dt, form, epi, M, N, K):
    rows = plan_rows(dt, form, epi, M, N, K)
    if rows:
        return rows
    n = 2 * N if epi == GATED else N
    stages = up(K, 128 // SIZE[dt])
    best, least = None, 0.0
    for kernel, (bm, bn, per_cu, stage, round_us) in TILES[dt].items():
        scale = 1.0
        if kernel == 64 and epi == GATED:
            bn, scale = 128, 1.8
        us = [0.0] + [scale * s for s in stage]
        tiles = up(M, bm) * up(n, bn)
        each = tiles // CUS
        last = each % per_cu
        time = (each // per_cu) * (stages * us[per_cu] + round_us)
        whole, splits = tiles, 1
        if tiles % (CUS * per_cu):
            tail = stages * us[last + 1 if tiles % CUS else last]
            for beside in sorted({0, last}):
                rest = tiles - (each - last + beside) * CUS
                if not rest:
                    continue
                free, before = per_cu - beside, 0
                for r in range(1, 4 * free + 1):
                    slices = min(r * CUS // rest, stages // 4)
                    if slices < 2 or slices == before:
                        continue
                    before = slices
                    per = up(stages, slices)
                    units = rest * up(stages, per)
                    u = up(units, CUS)
                    t = 3.0 + units * bm * bn * 4e-6 * 0.22
                    if u <= free:
                        t += stages * us[beside] + per * (us[beside + u] - us[beside])
                    else:
                        t += (beside * stages + up(u, free) * free * per) * us[per_cu] / per_cu
                    if t < tail:
                        tail, whole, splits = t, tiles - rest, up(stages, per)
            time += tail + round_us
        if best is None or time < least:
            least = time
            best = Plan(kernel, tiles, whole, splits,
                        align256((tiles - whole) * splits * bm * bn * 4))
    return best


def b(v):
    return "true" if v else "false"


def product(dt, form, epi, M, N, K, words=False):
    """{kernel: state} of one product with its epilogue. words: it has arrival words."""
    p, e = plan(dt, form, epi, M, N, K), NAME[dt]
    if p.kernel == "rows":
        rt = 1 if M <= 16 else 2 if M <= 32 else 4
        depth = 1 if rt == 4 else 2
        name = f"few_rows_kernel<{e}, {b(form == KT)}, %d, {rt}, {p.cols}, 8, {depth}>"
        if p.splits > 1 and not words:
            return {name % PARTIAL: "split", f"join_rows_kernel<{e}, {epi}>": "split"}
        return {name % epi: p.state}
    ab = f"{b(form == TT)}, {b(form != KK)}, {epi}"
    if p.kernel == 256:
        out = {f"big_kernel<{ab}>": p.state}
    else:
        tile = "64, 128, 2" if (p.kernel, epi) == (64, GATED) else \
            "64, 64, 3" if p.kernel == 64 else "128, 128, 2"
        out = {f"gemm_kernel<{e}, {ab}, {tile}>": p.state}
    if p.splits > 1:
        wave = {256: "2, 4, 4, 2", 128: "2, 2, 2, 2", 64: f"2, 2, 1, {2 if epi == GATED else 1}"}
        out[f"join_kernel<{e}, {epi}, {wave[p.kernel]}>"] = p.state
    return out


def merge(*parts):
    """kernel -> its states."""
    out = {}
    for part in parts:
        for k, state in part.items():
            out.setdefault(k, set()).update(state if isinstance(state, set) else {state})
    return out


def linear(dt, rows, k, n, transposed, act, bias, residual, train=True, captured=False):
    """The kernels of fused_linear, and of its backward pass for every operand. (Forward
    passes have arrival words, but captured ones.)"""
    parts = [product(dt, KK if transposed else KT, LINEAR, rows, n, k, not captured)]
    if train:
        if act or bias:
            slope = 0 if not act else 2 if act == "relu" and not residual else 1
            parts.append({f"act_grad_kernel<{NAME[dt]}, {slope}>": "whole"})
        if bias:
            parts.append({"col_sum_kernel": "whole"})
        parts.append(product(dt, KT if transposed else KK, LINEAR, rows, k, n))
        parts.append(product(dt, TT, LINEAR, *((n, k) if transposed else (k, n)), rows))
    return merge(*parts)


def gated(dt, rows, d, width, t1, t2, bias, train=True, captured=False):
    """The kernels of gated_mlp, and of its backward pass for every operand."""
    parts = [product(dt, KK if t1 else KT, GATED, rows, width, d, not captured),
             product(dt, KK if t2 else KT, LINEAR, rows, d, width, not captured)]
    if train:
        parts.append(product(dt, KT if t2 else KK, GATED_BWD, rows, width, d))
        if bias:
            parts.append({f"act_grad_kernel<{NAME[dt]}, 0>": "whole", "col_sum_kernel": "whole"})
        parts.append(product(dt, TT, LINEAR, *((d, width) if t2 else (width, d)), rows))
        parts.append(product(dt, KT if t1 else KK, LINEAR, rows, d, 2 * width))
        parts.append(product(dt, TT, LINEAR, *((2 * width, d) if t1 else (d, 2 * width)), rows))
    return merge(*parts)


def norm(dt, rows, d, aligned, weights, train=True):
    """The kernels of layer_norm over rows d apart (aligned: of whole chunks), and of its
    backward pass."""
    v = 16 // SIZE[dt]
    threads = next(t for t, most in ((8, 64), (16, 256), (64, 1024), (256, 4096), (1024, 16384))
                   if d <= most)
    head = f"{NAME[dt]}, {threads}, {(8 if d <= threads * 8 else 16) // v}, {b(aligned and d % v == 0)}"
    out = {f"norm_fwd_kernel<{head}>"}
    if train:
        out.add(f"norm_bwd_kernel<{head}, {b(weights)}>")
        if weights:
            out.add("col_sum_kernel")
    return {k: {"whole"} for k in out}


KERNEL = re.compile(r"\b((?:big|gemm|join|few_rows|join_rows|act_grad|norm_fwd|norm_bwd)_kernel"
                    r"<[^()]*>|col_sum_kernel)")


def plain_name(symbol):
    """A kernel's name without namespaces and arguments, or None. (The expert layer's
    products have kernels of other names or other template arguments.)"""
    symbol = re.sub(r"vmoe::|dense::|\(anonymous namespace\)::", "", symbol).replace("(SlopeOf)", "")
    symbol = re.sub(r"\((?:SlopeOf|int)\)", "", symbol)
    m = KERNEL.search(symbol)
    return m and m.group(1)


def library_kernels(path):
    """The dense operators' kernels that the library holds (its own symbol table)."""
    out = subprocess.run(["nm", "-C", "--defined-only", str(path)], check=True,
                         capture_output=True, text=True).stdout
    return {n for n in (plain_name(line) for line in out.splitlines()
                        if "dense::" in line or "norm_" in line or "col_sum" in line) if n}

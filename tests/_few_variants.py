"""Which kernels of csrc/few_tokens.hip a call takes: its launch rules, written
down a second time, so that tests can be shown to reach every kernel the library
holds. The GPU tests hold these rules to the kernels that run."""

from __future__ import annotations

import re
import subprocess


def up(a, b):
    return -(-a // b)


def split_waves(steps):
    wk = 1
    while wk < 8 and wk < steps:
        wk *= 2
    return wk


# weights -> (name, columns of a wave's tile)
def bf16(cpl):
    return f"WBf16<{cpl}>", 16 * cpl


def f32(cpl):
    return f"WF32<{cpl}>", 16 * cpl


def q4(blocks, group):
    return f"WQ4<{blocks}, {group // 32}>", 16 * blocks


UP, DOWN, PLAIN = 0, 1, 2


def kernel(w, mode, mt, ns, slot, depth, early):
    b = ("false", "true")
    return f"few_kernel<{w[0]}, {mode}, {mt}, {ns}, {b[slot]}, {depth}, {b[early]}>"


def by_expert(w, mode, ns, depth, wk, pairs, E, tiles1, cols, rows=None):
    """launch(): a workgroup takes an expert and a column tile."""
    four = w[0].startswith("WQ4")
    if rows is None:
        rows = 2 * pairs // E
    mt = 1
    if (not four or mode == PLAIN) and rows > 16:
        mt, depth = 2, 1
    width = 8 // wk * w[1]
    units = tiles1 * 64 // width if mode == UP else E * up(cols, width)
    early = pairs >= E and (not four or units <= 512)
    return kernel(w, mode, mt, ns, False, depth, early)


def layer_kernels(dt, group, d, widths, k, T, act="relu_squared", router=True):
    """The kernels of moe_few_tokens (experts_few_tokens: router=False)."""
    E, pairs, ns, wide = len(widths), T * k, 2 if act == "swiglu" else 1, max(widths)
    tiles1 = sum(up(w, 64) for w in widths)
    small = pairs * 4 <= E or pairs * (tiles1 * 64 / E) * d <= (1 << 23 if dt == "f32" else 1 << 24)
    slots = small and pairs * 2 <= E and E <= 256
    out = {f"few_logits_kernel<{'true' if dt == 'f32' else 'false'}>"} if router else set()

    steps = up(d, {"bf16": 32, "f32": 16, "q4": 128}[dt])
    if slots:
        units = pairs * up(wide, 64)
        if dt == "bf16":
            w, depth = (bf16(4), 4 // ns) if units >= 256 else (bf16(2), 4)
        elif dt == "f32":
            w, depth = f32(2), 4
        else:
            w, depth = (q4(4 // ns, group), 1) if units >= 128 else (q4(1, group), 2)
        out.add(kernel(w, UP, 1, ns, True, depth, False))
    else:
        wk = 8
        if dt == "q4":
            if steps > 4 and tiles1 < 256:
                w = q4(2, group)
            elif steps > 4 and ns == 1:
                w = q4(4, group)
            else:
                w, wk = q4(2, group), 4
        else:
            cpl = 2 if tiles1 < 256 else 4
            w = f32(cpl) if dt == "f32" else bf16(cpl)
        out.add(by_expert(w, UP, ns, 1, wk, pairs, E, tiles1, wide))
    if small:
        token = {"bf16": ("WBf16<2>", 4), "f32": ("WF32<2>", 4)}.get(dt, (q4(1, group)[0], 2))
        out.add(f"few_token_kernel<{token[0]}, {token[1]}, {'false' if slots else 'true'}>")
        return out

    steps = up(wide, {"bf16": 32, "f32": 16, "q4": 128}[dt])
    wk, depth = split_waves(steps), 1
    if dt == "q4":
        w = q4(4 if E * up(d, 8 // wk * 64) >= 256 else 2, group)
    elif dt == "f32":
        w = f32(4)
    else:
        w = bf16(4)
        if steps <= 8:
            wk, depth = split_waves(up(steps, 2)), 2
    out.add(by_expert(w, DOWN, 1, depth, wk, pairs, E, tiles1, d))
    out.add("few_combine_kernel")
    return out


def matvec_kernels(group, K, lengths, k, T):
    """The kernels of matvec_q4; k = 0: without ids."""
    w, cols = q4(2, group), max(lengths)
    wk = split_waves(up(K, 128))
    return {by_expert(w, PLAIN, 1, 1, wk, T * max(k, 1), len(lengths), 0, cols,
                      rows=None if k else T)}


def plain_name(symbol):
    """A kernel's name without namespaces and arguments, or None."""
    symbol = re.sub(r"vmoe::|\(anonymous namespace\)::", "", symbol).replace("(Mode)", "")
    m = re.search(r"\b(few_(?:kernel|token_kernel|logits_kernel)<[^()]*>|few_combine_kernel)", symbol)
    return m and m.group(1)


def library_kernels(path):
    """The few-token kernels that the library holds (its own symbol table)."""
    out = subprocess.run(["nm", "-C", "--defined-only", str(path)], check=True,
                         capture_output=True, text=True).stdout
    return {n for n in map(plain_name, out.splitlines()) if n}

"""Calls of the dense operators that are settled on the host."""

from __future__ import annotations

import os
import shutil
import subprocess
import sys

import pytest
import torch

from triton_moe import _lib
from triton_moe import kernels as K


class Wrapper(torch.Tensor):
    """A tensor whose values are in another one, as a distributed tensor's are."""

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, strides=inner.stride(),
                                                   dtype=inner.dtype, device=inner.device)

    def __init__(self, inner):
        self.inner = inner

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        args = [a.inner if isinstance(a, Wrapper) else a for a in args]
        return func(*args, **(kwargs or {}))


def freed(t):
    t = t.clone(memory_format=torch.contiguous_format)
    t.untyped_storage().resize_(0)
    return t


def freed_slice(t):
    """(its address is not 0)"""
    flat = torch.zeros(t.numel() + 64, dtype=t.dtype, device=t.device)
    out = flat[64:].view(t.shape)
    flat.untyped_storage().resize_(0)
    return out


def cut(t):
    t = t.clone(memory_format=torch.contiguous_format)
    t.untyped_storage().resize_(t.numel() * t.element_size() - 1)
    return t


WITHOUT_MEMORY = [Wrapper, freed, freed_slice, cut]


def calls(x, w, v, of):
    """(operand, call) with one operand as `of` gives it; w [8, 8], v [8]."""
    wide, w2, v2 = torch.cat([w, w], 1), w, torch.cat([v, v])
    return [("weight", lambda: K.layer_norm(x, of(v), v)), ("bias", lambda: K.layer_norm(x, v, of(v))),
            ("weight", lambda: K.fused_linear(x, of(w))), ("bias", lambda: K.fused_linear(x, w, of(v))),
            ("residual", lambda: K.fused_linear(x, w, v, "relu", of(x))),
            ("w1", lambda: K.gated_mlp(x, of(wide), w2)), ("w2", lambda: K.gated_mlp(x, wide, of(w2))),
            ("bias1", lambda: K.gated_mlp(x, wide, w2, bias1=of(v2))),
            ("bias2", lambda: K.gated_mlp(x, wide, w2, bias2=of(v))),
            ("residual", lambda: K.gated_mlp(x, wide, w2, residual=of(x)))]


@pytest.mark.parametrize("of", WITHOUT_MEMORY)
def test_operands_without_memory(of):
    """An operand whose values are elsewhere, or gone, is refused: it does not count as
    not given."""
    for what, call in calls(torch.zeros(3, 8), torch.zeros(8, 8), torch.zeros(8), of):
        with pytest.raises(NotImplementedError, match=f"{what} has no memory"):
            call()


def run_python(code, **env):
    return subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                          env={**os.environ, **env})


def test_library_of_another_place(tmp_path):
    """VMOE_LIB names the one library of the process: the dense operators call it too, and
    need none in the package's directory."""
    package = tmp_path / "package" / "triton_moe"
    here = _lib.LIB_PATH.parent
    shutil.copytree(here, package, ignore=shutil.ignore_patterns("libvmoe.so", "__pycache__"))
    library = tmp_path / "elsewhere.so"
    shutil.copy(_lib.LIB_PATH, library)
    for path in (package.parent, here.parent):
        out = run_python("import sys; sys.path.insert(0, %r)\n"
                         "from triton_moe import _lib, kernels\n"
                         "import torch\n"
                         "_lib.dense()\n"
                         "try: kernels.layer_norm(torch.zeros(1, kernels.layer_norm_max() + 1))\n"
                         "except NotImplementedError as e: print(e)\n"
                         "names = {l.split()[-1] for l in open('/proc/self/maps') if '/' in l}\n"
                         "print(sorted(n for n in names if 'vmoe' in n or 'elsewhere' in n))\n"
                         % str(path), VMOE_LIB=str(library))
        assert out.returncode == 0, out.stderr
        assert "rows of at most 16384" in out.stdout
        assert out.stdout.strip().endswith(f"['{library}']"), out.stdout


def test_module_without_a_library():
    """The extension module by itself calls nothing."""
    out = run_python("import sys, torch; sys.path.insert(0, %r)\n"
                     "from triton_moe import _dense\n"
                     "try: _dense.layer_norm(torch.zeros(1, 8), None, None, 1e-5)\n"
                     "except RuntimeError as e: print(e)\n"
                     "try: _dense.use(0)\n"
                     "except RuntimeError as e: print(e)\n" % str(_lib.LIB_PATH.parent.parent))
    assert out.returncode == 0 and out.stdout.count("library") == 2, out.stdout + out.stderr


def test_what_a_backward_pass_does_not_read_is_not_asked_for():
    """At the C entry points (no call here reaches a launch: the workspace is short)."""
    lib, p, short = _lib.lib(), 0x1000, _lib.ERR_WORKSPACE

    def gated(x=None, w1=None, w2=None, h=None, z=None, gx=None, gw1=None, gb1=None, gw2=None, gb2=None):
        return lib.vmoe_gated_backward(0, p, 64, x, 64, 2, 64, 32, w1, 64, 0, w2, 64, 0, 3, h, z, gx, 64,
                                       gw1, 64, gb1, 0, gw2, 64, gb2, 0, p, 0, None)
    assert gated(gb2=p) == short
    assert gated(h=p, gw2=p) == short
    assert gated(w2=p, z=p, gb1=p) == short
    assert gated(x=p, w2=p, z=p, gw1=p) == short
    assert gated(w1=p, w2=p, z=p, gx=p) == short
    for lacks in (dict(gw2=p), dict(z=p, gb1=p), dict(w2=p, gb1=p), dict(w2=p, z=p, gw1=p),
                  dict(w2=p, z=p, gx=p), dict(w1=p, z=p, gx=p)):
        assert gated(**lacks) == _lib.ERR_INVALID_ARG

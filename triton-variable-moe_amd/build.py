"""Builds libvmoe.so (the gfx950 HIP kernels behind include/vmoe.h) and _dense.so (the
extension module that calls the dense operators of it from torch).

Usage: python triton-variable-moe_amd/build.py [--jobs N]

Both are written into the Python package (triton_moe/) so that it finds them without
an install step. libvmoe.so needs hipcc alone; without torch's headers or a C++ compiler
it is built without the extension module.
"""

from __future__ import annotations

import argparse
import concurrent.futures as cf
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

HERE = Path(__file__).resolve().parent
REPO = HERE.parent
CSRC = HERE / "csrc"
OUT = HERE / "triton_moe" / "libvmoe.so"
DENSE = HERE / "triton_moe" / "_dense.so"
OBJ = HERE / "_build"
SOURCES = ["route.hip", "permute.hip", "permute_f32.hip", "gemm.hip", "gemm_few_rows.hip",
           "gemm_f32.hip", "router.hip", "router_bwd.hip", "expert.hip", "expert_f32.hip",
           "few_tokens.hip", "few_q4.hip", "dense.hip", "dense_gemm.hip", "dense_big.hip",
           "dense_few.hip", "norm.hip", "capi.hip"]

HIPCC_FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-Wall",
    "-Wno-unused-function",
    f"-I{REPO / 'include'}",
    f"-I{CSRC}",
    # No packed-fp32 instructions in device code (they have given silent
    # wrong results on this hardware pool); the host pass ignores the flag.
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("hipcc not found (set HIPCC or install ROCm)")


def _compile(src: str) -> Path:
    obj = OBJ / (Path(src).stem + ".o")
    cmd = [hipcc(), *HIPCC_FLAGS, "-c", str(CSRC / src), "-o", str(obj)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{res.stdout}\n{res.stderr}")
    return obj


def _torch_dir() -> Path:
    spec = importlib.util.find_spec("torch")  # (found, not imported)
    if spec is None or spec.origin is None:
        raise RuntimeError("torch not found")
    return Path(spec.origin).parent


def _dense_lacks() -> str | None:
    """What the extension module would need and is not there."""
    compiler = os.environ.get("CXX", "g++")
    if shutil.which(compiler) is None:
        return f"no C++ compiler ({compiler})"
    try:
        torch = _torch_dir()
    except RuntimeError as exc:
        return str(exc)
    for header in (torch / "include/ATen/ATen.h", Path(sysconfig.get_paths()["include"]) / "Python.h"):
        if not header.exists():
            return f"no {header}"
    return None


def _compile_dense() -> Path:
    """The extension module that calls the dense operators: host code alone, with
    torch's headers."""
    torch = _torch_dir()
    obj = OBJ / "dense_torch.o"
    rocm = Path(hipcc()).resolve().parents[1]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-Wall",
           "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1", f"-I{REPO / 'include'}",
           "-isystem", str(torch / "include"),
           "-isystem", str(torch / "include/torch/csrc/api/include"),
           "-isystem", sysconfig.get_paths()["include"], "-isystem", str(rocm / "include"),
           "-c", str(CSRC / "dense_torch.cpp"), "-o", str(obj)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed for dense_torch.cpp:\n{res.stdout}\n{res.stderr}")
    return obj


def _link_dense(obj: Path) -> None:
    tmp = DENSE.with_suffix(".so.tmp")
    cmd = [os.environ.get("CXX", "g++"), "-shared", str(obj), "-o", str(tmp),
           f"-L{_torch_dir() / 'lib'}", "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_python", "-ldl"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, DENSE)


def build(jobs: int = 4, verbose: bool = False) -> Path:
    OBJ.mkdir(parents=True, exist_ok=True)
    lacks = _dense_lacks()
    with cf.ThreadPoolExecutor(max_workers=max(1, jobs)) as ex:
        dense = None if lacks else ex.submit(_compile_dense)
        objs = list(ex.map(_compile, SOURCES))
    tmp = OUT.with_suffix(".so.tmp")
    cmd = [hipcc(), "--offload-arch=gfx950", "-shared", "-fPIC", *map(str, objs), "-o", str(tmp)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, OUT)
    if dense:
        _link_dense(dense.result())
    else:
        DENSE.unlink(missing_ok=True)  # (of an earlier build)
        print(f"{DENSE.name} is not built: {lacks}; the dense operators need it",
              file=sys.stderr)
    if verbose:
        print(f"built {OUT}" + (f", {DENSE}" if dense else ""))
    return OUT


def main() -> int:
    ap = argparse.ArgumentParser()
    ap.add_argument("--jobs", type=int, default=4)
    args = ap.parse_args()
    build(args.jobs, verbose=True)
    return 0


if __name__ == "__main__":
    sys.exit(main())

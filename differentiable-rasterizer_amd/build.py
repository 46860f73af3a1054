"""Builds libdiffrast_hip.so (gfx950) in-tree with hipcc, and the native torch
operations of diffrast.layers over it with the host compiler.

Usage: python build.py [--verbose]. The library lands next to this file, where
`diffrast._lib` loads it from, the torch operations in diffrast/.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
ROOT = HERE.parent
CSRC = HERE / "csrc"
LIB = HERE / "libdiffrast_hip.so"
TORCH_SOURCE = CSRC / "torch_layers.cpp"
TORCH_LIB = HERE / "diffrast" / "_torch_layers.so"
ARCH = os.environ.get("DIFFRAST_OFFLOAD_ARCH", "gfx950")

SOURCES = [CSRC / "kernels.hip", CSRC / "runtime.hip", CSRC / "fit.hip", CSRC / "scratch.hip", CSRC / "resize.hip",
           CSRC / "layers.hip", CSRC / "layer_norm.hip", CSRC / "linear.hip", CSRC / "dropout.hip",
           CSRC / "rms_norm.hip", CSRC / "gated.hip", CSRC / "linear8.hip", CSRC / "adamw.hip"]

# -ffp-contract=off: the kernels state every FMA explicitly; plain a*b+c must
# round twice, as the reference's arithmetic does.
# -packed-fp32-ops: no v_pk_*_f32 instructions in the generated code.
# -structurizecfg-skip-uniform-regions: regions whose branches are all
# wave-uniform (scalar-condition branches) keep their control flow as written;
# the default structurizer rewrites them as it does divergent ones, carrying
# path flags (scalar mask operations and extra branches) through the sweeps'
# per-entry code. Regions with a divergent branch are structurized as before.
FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-ffp-contract=off",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-mllvm", "-structurizecfg-skip-uniform-regions=true",
    "-Wall",
    f"-I{ROOT / 'include'}",
    f"-I{CSRC}",
]


def hipcc() -> str:
    for cand in (shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("hipcc not found")


def _run(cmd: list[str], verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    noise = "packed-fp32-ops"
    err = "\n".join(l for l in (res.stderr or "").splitlines() if noise not in l)
    if res.returncode != 0:
        raise RuntimeError(f"{Path(cmd[0]).name} failed ({res.returncode}):\n{err}")
    if verbose and err.strip():
        print(err)


def build(verbose: bool = False) -> Path:
    """Compiles each source (several at a time), then links them."""
    cc, tmp = hipcc(), LIB.with_suffix(".so.tmp")
    with tempfile.TemporaryDirectory() as objdir:
        objs = [str(Path(objdir) / f"{src.stem}.o") for src in SOURCES]
        with ThreadPoolExecutor(min(4, os.cpu_count() or 1)) as pool:
            list(pool.map(lambda so: _run([cc, *FLAGS, "-c", str(so[0]), "-o", so[1]], verbose), zip(SOURCES, objs)))
        _run([cc, f"--offload-arch={ARCH}", "-fPIC", "-shared", *objs, "-o", str(tmp)], verbose)
    os.replace(tmp, LIB)
    return LIB


def build_torch(verbose: bool = False) -> Path | None:
    """The native torch operations (host code alone), linked to LIB; None without PyTorch."""
    try:
        import torch
    except ImportError:
        return None
    pkg = Path(torch.__file__).resolve().parent
    rocm = Path(hipcc()).resolve().parents[1]
    tmp = TORCH_LIB.with_suffix(".so.tmp")
    _run([shutil.which("g++") or "c++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-Wno-sign-compare",
          "-Wno-unknown-pragmas", "-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM", "-DTORCH_EXTENSION_NAME=_torch_layers",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
          *(f"-isystem{d}" for d in (pkg / "include", pkg / "include" / "torch" / "csrc" / "api" / "include",
                                     rocm / "include", sysconfig.get_paths()["include"])),
          f"-I{ROOT / 'include'}", str(TORCH_SOURCE), "-o", str(tmp), f"-L{pkg / 'lib'}", f"-L{HERE}",
          "-ltorch", "-ltorch_cpu", "-ltorch_hip", "-lc10", "-lc10_hip", "-ltorch_python", "-ldiffrast_hip",
          "-Wl,-rpath,$ORIGIN/.."], verbose)
    os.replace(tmp, TORCH_LIB)
    return TORCH_LIB


if __name__ == "__main__":
    print(build(verbose="--verbose" in sys.argv))
    print(build_torch(verbose="--verbose" in sys.argv))

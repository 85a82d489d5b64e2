"""Builds ``libbioemu2_mi355x.so`` (all HIP kernels + the C ABI) and ``libbioemu2_torch.so`` (the trainable operators
as torch ops over it) in-tree for gfx950.

Usage: ``python -m bioemu2_amd.build`` (also called by ``__graft_entry__.build()``).
Always recompiles; both ``.so`` land next to this file so they travel with the
source tree and are what the Python layer loads.
"""

from __future__ import annotations

import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import tempfile
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
CSRC = PKG_DIR / "csrc"
INCLUDE = PKG_DIR.parent / "include"
LIB_NAME = "libbioemu2_mi355x.so"
TORCH_LIB_NAME = "libbioemu2_torch.so"
ARCH = os.environ.get("BIOEMU_OFFLOAD_ARCH", "gfx950")

# Packed-fp32 VALU ops are disabled for device code; the host pass warns that
# it does not know the feature, which is harmless.
# -fno-honor-nans: lets fmaxf lower to a single v_max_f32 instead of
# canonicalise + max.  Infinities are still honoured (the softmax masks use
# -inf); a kernel that has to tell a NaN apart does so on its bits
# (sigmoid_ulp), because the compiler may fold comparisons with one.
# -amdgpu-mfma-vgpr-form: MFMA accumulators live in VGPRs, which removes the
# AGPR<->VGPR copies around every softmax / epilogue touch of an accumulator.
HIPCC_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-Wall",
    "-Wno-unused-function",
    "-Xclang",
    "-target-feature",
    "-Xclang",
    "-packed-fp32-ops",
    "-fno-honor-nans",
    "-mllvm",
    "-amdgpu-mfma-vgpr-form",
    f"-I{INCLUDE}",
]


def _hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("hipcc not found (set HIPCC or install ROCm)")


def _compile(src: Path, obj: Path) -> None:
    cmd = [_hipcc(), *HIPCC_FLAGS, "-c", str(src), "-o", str(obj)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    out = "\n".join(
        ln for ln in (res.stdout + res.stderr).splitlines() if "packed-fp32-ops" not in ln
    )
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src.name}:\n{out}")
    if out.strip():
        print(out, file=sys.stderr)


def _compile_torch(obj: Path) -> None:
    """The torch ops' glue: host code against the installed torch."""
    import torch
    from torch.utils.cpp_extension import include_paths

    rocm = Path(_hipcc()).resolve().parents[1]
    cmd = [
        shutil.which("g++") or _hipcc(), "-O2", "-std=c++17", "-fPIC", "-Wall", "-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM",
        f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
        *(f"-isystem{p}" for p in include_paths()), f"-isystem{rocm / 'include'}", f"-I{INCLUDE}",
        "-c", str(CSRC / "torch_ops.cpp"), "-o", str(obj),
    ]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed for torch_ops.cpp:\n{res.stdout}{res.stderr}")


def _install(built: Path, name: str) -> Path:
    """Atomic replace, so that a running process never maps a half-written file."""
    target = PKG_DIR / name
    staged = target.with_suffix(".so.tmp")
    shutil.copy2(built, staged)
    os.replace(staged, target)
    return target


def _link(cmd: list[str]) -> None:
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}{res.stderr}")


def build(verbose: bool = True) -> Path:
    sources = sorted(CSRC.glob("*.hip"))
    if not sources:
        raise RuntimeError(f"no HIP sources under {CSRC}")
    with tempfile.TemporaryDirectory(prefix="bioemu_build_") as tmp:
        objs = [Path(tmp) / (s.stem + ".o") for s in sources]
        glue = Path(tmp) / "torch_ops.o"
        with cf.ThreadPoolExecutor(max_workers=min(8, len(sources) + 1)) as ex:
            torch_done = ex.submit(_compile_torch, glue)   # the longest, first
            list(ex.map(_compile, sources, objs))
            torch_done.result()
        tmp_lib, tmp_torch = Path(tmp) / LIB_NAME, Path(tmp) / TORCH_LIB_NAME
        _link([_hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", *map(str, objs), "-o", str(tmp_lib)])
        import torch

        torch_lib = Path(torch.__file__).resolve().parent / "lib"
        _link([shutil.which("g++") or _hipcc(), "-shared", "-fPIC", str(glue), "-o", str(tmp_torch), f"-L{tmp}",
               f"-l:{LIB_NAME}", f"-L{torch_lib}", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_hip", "-Wl,-rpath,$ORIGIN"])
        target = _install(tmp_lib, LIB_NAME)
        _install(tmp_torch, TORCH_LIB_NAME)
    if verbose:
        print(f"built {target} from {len(sources)} sources for {ARCH}, and {TORCH_LIB_NAME}")
    return target


if __name__ == "__main__":
    build()

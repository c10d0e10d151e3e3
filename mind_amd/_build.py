"""Build the gfx950 HIP library ``mind_amd/lib/libesa_hip.so`` and the host module ``mind_amd/lib/esa_tensors.so``.

Each ``csrc/*.hip`` file is compiled to an object with ``hipcc
--offload-arch=gfx950`` (in parallel), then linked into one shared library
whose only exported symbols are the ``extern "C"`` entry points declared in
``include/esa_hip.h``.  Objects go to ``mind_amd/_build/`` and stay out of
version control; the ``.so`` is built in-tree so it travels with the
tree.  ``csrc/esa_tensors.cpp`` (reading lists of
torch tensors) is host code against torch's and Python's headers.
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
LIBDIR = PKG / "lib"
LIB = LIBDIR / "libesa_hip.so"
TENSORS = LIBDIR / "esa_tensors.so"
INCLUDE = PKG.parent / "include"

ARCH = "gfx950"
# Packed fp32 VALU ops (v_pk_*_f32) are disabled for all device code: some of
# their forms have given wrong results on the target machines.  The host pass
# warns that it does not know the feature; that is harmless.
HIPFLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    # MFMA accumulators in ordinary VGPRs (no AGPR copies around the softmax).
    "-mllvm", "-amdgpu-mfma-vgpr-form=true",
    "-fvisibility=hidden",
    f"-I{INCLUDE}",
]


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("hipcc not found: the MI355X library cannot be built")


def _compile(src: Path) -> Path:
    obj = BUILD / (src.stem + ".o")
    cmd = [hipcc(), *HIPFLAGS, "-c", str(src), "-o", str(obj)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        msg = "\n".join(line for line in proc.stderr.splitlines() if "packed-fp32-ops" not in line)
        raise RuntimeError(f"hipcc failed on {src.name}:\n{msg}")
    return obj


def _build_tensors() -> None:
    import torch
    from torch.utils.cpp_extension import include_paths, library_paths
    src, tmp = CSRC / "esa_tensors.cpp", TENSORS.with_suffix(".so.tmp")
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", f"-I{sysconfig.get_paths()['include']}",
           *(f"-I{p}" for p in include_paths()), f"-I{Path(hipcc()).resolve().parent.parent / 'include'}",
           "-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM", str(src), "-o", str(tmp), *(f"-L{p}" for p in library_paths()),
           "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_hip"]   # torch has loaded them by the time this module is
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"g++ failed on {src.name}:\n{proc.stderr}")
    os.replace(tmp, TENSORS)


def build(verbose: bool = True) -> Path:
    """Compile every source; link ``libesa_hip.so`` and ``esa_tensors.so``.  Always rebuilds."""
    BUILD.mkdir(exist_ok=True)
    LIBDIR.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.hip"))
    if not sources:
        raise RuntimeError(f"no HIP sources under {CSRC}")
    with cf.ThreadPoolExecutor(max_workers=min(8, len(sources) + 1)) as ex:
        tensors = ex.submit(_build_tensors)
        objs = list(ex.map(_compile, sources))
        tensors.result()
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", *map(str, objs), "-o", str(tmp)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"link of {LIB.name} failed:\n{proc.stderr}")
    os.replace(tmp, LIB)
    if verbose:
        print(f"[mind_amd] built {LIB} from {len(sources)} HIP sources, and {TENSORS}", file=sys.stderr)
    return LIB


if __name__ == "__main__":
    build()

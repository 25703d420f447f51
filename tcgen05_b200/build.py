"""Build the emulator's CUDA library (sm_100a) in-tree.

``python -m tcgen05_b200.build`` compiles every ``csrc/*.cu`` into
``tcgen05_b200/_lib/libt5e.so`` with nvcc, for the B200 architecture only
(``-gencode arch=compute_100a,code=sm_100a``).  The library links the CUDA
runtime statically, so loading it needs no GPU and no CUDA library path.
``csrc/t5e_torch.cpp`` becomes ``_lib/t5e_torch.so``, the PyTorch side of the
block-scaled calls, against the installed PyTorch and that library.
"""

from __future__ import annotations

import os
import shlex
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
LIB_DIR = PKG / "_lib"
LIB = LIB_DIR / "libt5e.so"
TORCH_SRC = CSRC / "t5e_torch.cpp"
TORCH_LIB = LIB_DIR / "t5e_torch.so"
INCLUDE = ROOT / "include"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC,-O2"]


def nvcc() -> str:
    found = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(found).exists():
        raise RuntimeError("nvcc not found; the emulator needs the CUDA toolkit to build")
    return found


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def build_torch(verbose: bool = False, force: bool = False) -> Path | None:
    """Compile the PyTorch side if its sources are newer or it was built for
    another PyTorch or Python; return its path.  Without PyTorch or a C++
    compiler it is left out, with a message: the C ABI needs neither."""
    import sysconfig

    try:
        import torch
    except ImportError as e:
        print(f"{TORCH_LIB.name} is left out: {e}", file=sys.stderr, flush=True)
        return None
    cxx = shlex.split(os.environ.get("CXX") or "g++")  # $CXX may hold a wrapper and options
    if shutil.which(cxx[0]) is None:
        print(f"{TORCH_LIB.name} is left out: no C++ compiler {cxx[0]}", file=sys.stderr, flush=True)
        return None
    built_for = f"torch {torch.__version__} python {sys.version_info[0]}.{sys.version_info[1]}"
    deps = [TORCH_SRC, INCLUDE / "t5e.h"]
    # the library holds the words it was built with
    if not force and TORCH_LIB.exists() and all(TORCH_LIB.stat().st_mtime >= p.stat().st_mtime for p in deps) \
            and f"t5e_torch for {built_for}\0".encode() in TORCH_LIB.read_bytes():
        return TORCH_LIB
    cuda = Path(nvcc()).resolve().parents[1] / "include"
    home = Path(torch.__file__).resolve().parent
    includes = [INCLUDE, sysconfig.get_paths()["include"], cuda, home / "include", home / "include/torch/csrc/api/include"]
    tmp = TORCH_LIB.with_suffix(".so.tmp")
    cmd = [*cxx, "-O2", "-std=c++17", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-DTORCH_EXTENSION_NAME=t5e_torch",
           f'-DT5E_BUILT_FOR="t5e_torch for {built_for}"',
           *[arg for i in includes for arg in ("-isystem", str(i))], str(TORCH_SRC), "-o", str(tmp),
           "-L", str(LIB_DIR), "-l:libt5e.so", "-L", str(home / "lib"), "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu",
           "-ltorch_python",
           # PyTorch's C++ library, whatever $CXX links by itself: a static copy has locale facets of its own, and the
           # first message that a refused call prints through libc10 ends the process
           "-nostdlib++", "-l:libstdc++.so.6", "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, TORCH_LIB)
    return TORCH_LIB


def build(verbose: bool = False, ptxas_info: bool = False, force: bool = False) -> Path:
    """Compile the libraries whose sources are newer than they are; return the
    CUDA library's path."""
    path = _build_cuda(verbose, ptxas_info, force)
    build_torch(verbose, force)
    return path


def _build_cuda(verbose: bool, ptxas_info: bool, force: bool) -> Path:
    LIB_DIR.mkdir(exist_ok=True)
    srcs = sources()
    deps = srcs + sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + [INCLUDE / "t5e.h"]
    if not force and LIB.exists() and all(LIB.stat().st_mtime >= p.stat().st_mtime for p in deps):
        return LIB
    objs = []
    obj_dir = LIB_DIR / "obj"
    obj_dir.mkdir(exist_ok=True)
    extra = ["-Xptxas", "-v"] if ptxas_info else []
    for src in srcs:
        obj = obj_dir / (src.stem + ".o")
        cmd = [nvcc(), *ARCH, *NVCC_FLAGS, *extra, "-I", str(INCLUDE), "-I", str(CSRC), "-c", str(src), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
        objs.append(str(obj))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [nvcc(), *ARCH, "-shared", "-o", str(tmp), *objs]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    args = set(sys.argv[1:])
    print(build(verbose=True, ptxas_info="--ptxas-info" in args, force="--force" in args))

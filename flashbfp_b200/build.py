"""Build libflashbfp.so (sm_100a) in-tree with nvcc, and the Python module _fp8_bind with g++.

    python -m flashbfp_b200.build          # or flashbfp_b200.build.build()

Both land next to this file so that they travel with the source tree.
"""
from __future__ import annotations

import glob
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libflashbfp.so")
BIND = os.path.join(HERE, "_fp8_bind.so")
BIND_SOURCES = [os.path.join(CSRC, f) for f in ("fp8_bind.cpp", "attn_bind.cpp")]
BIND_STAMP = os.path.join(HERE, "_build", "fp8_bind.stamp")      # what BIND was built for
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-O3",
         "--expt-relaxed-constexpr", "-Xptxas", "-warn-spills"]


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _stale() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = sources() + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h"))
    deps += glob.glob(os.path.join(os.path.dirname(HERE), "include", "*.h"))
    return any(os.path.getmtime(p) > t for p in deps)


def bind_for() -> str:
    """What _fp8_bind.so is built for: another torch or Python needs another build."""
    try:
        version = importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:
        import torch
        version = torch.__version__
    return f"torch {version}, Python {sys.version_info[0]}.{sys.version_info[1]}"


def _bind_missing() -> str | None:
    """What this machine lacks to build _fp8_bind.so, if anything."""
    if importlib.util.find_spec("torch") is None:
        return "torch is not installed"
    if shutil.which("g++") is None:
        return "g++ is not installed"
    if not os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        return "Python.h is not installed"
    return None


def _bind_stale() -> bool:
    if not os.path.exists(BIND) or not os.path.exists(BIND_STAMP):
        return True
    deps = (*BIND_SOURCES, os.path.join(CSRC, "bind.h"), os.path.join(os.path.dirname(HERE), "include", "flashbfp.h"))
    if any(os.path.getmtime(p) > os.path.getmtime(BIND) for p in deps):
        return True
    with open(BIND_STAMP) as f:
        return f.read() != bind_for()


def _build_bind(force: bool, verbose: bool) -> None:
    """_fp8_bind.so: the Python entry points that check their tensors and call the library. The
    library alone (the C ABI) needs none of what this one needs, so a machine without it gets the
    library and a note; flashbfp_b200.fp8, .attention and .kv4 then say that the module is missing."""
    missing = _bind_missing()
    if not force and (missing is None or "torch" not in missing) and not _bind_stale():
        return
    if missing:
        print(f"{os.path.basename(BIND)} (the Python entry points of the 8-bit linears, the prompts' attention and the 4-bit cache) is not built: {missing}",
              file=sys.stderr, flush=True)
        return
    root = os.path.dirname(importlib.util.find_spec("torch").origin)
    import torch
    inc = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
           os.path.join(os.path.dirname(os.path.dirname(NVCC)), "include"), sysconfig.get_paths()["include"]]
    tmp = BIND + ".tmp"
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f'-DFBFP_BUILT_FOR="{bind_for()}"',
           *[a for i in inc for a in ("-isystem", i)], *BIND_SOURCES, "-o", tmp, "-L" + HERE,
           "-l:libflashbfp.so", "-L" + os.path.join(root, "lib"), "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10",
           "-lc10_cuda", "-Wl,-rpath,$ORIGIN", "-Wl,-rpath," + os.path.join(root, "lib")]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, BIND)
    os.makedirs(os.path.dirname(BIND_STAMP), exist_ok=True)
    with open(BIND_STAMP, "w") as f:
        f.write(bind_for())


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not _stale():
        _build_bind(force, verbose)
        return LIB
    objdir = os.path.join(HERE, "_build")
    os.makedirs(objdir, exist_ok=True)
    objs = []
    for src in sources():
        obj = os.path.join(objdir, os.path.basename(src)[:-3] + ".o")
        cmd = [NVCC, *ARCH, *FLAGS, "-c", src, "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
        objs.append(obj)
    tmp = LIB + ".tmp"
    cmd = [NVCC, *ARCH, "-shared", "-o", tmp, *objs, "-lcublasLt", "-Xlinker",
           "-rpath=" + os.path.join(os.path.dirname(os.path.dirname(NVCC)), "lib64")]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB)
    _build_bind(force, verbose)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))

"""Build recipe of libltm_b200.so: every csrc/*.cu compiled for sm_100a with
nvcc and linked into ltm_b200/libltm_b200.so (in-tree, so it travels with the
repository snapshot), and of ltm_b200/_torch_ops.so, the tensor-level callers of
its per-token operators (binding/torch_ops.cpp, g++ against PyTorch's headers; left
out, with a message, where there is no PyTorch: the C ABI does not need it).
Incremental: an object is rebuilt when its source or any header under csrc/ or
include/ is newer, _torch_ops.so also when it was built for another PyTorch or
Python (_build/torch_ops.for).

    python obsidian-memory-transformer_b200/build.py [--force] [-j N]
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
LIB = PKG / "ltm_b200" / "libltm_b200.so"
OPS_SRC = PKG / "binding" / "torch_ops.cpp"
OPS = PKG / "ltm_b200" / "_torch_ops.so"
OPS_FOR = BUILD / "torch_ops.for"  # what OPS was built for

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH + [
    "-O3", "-std=c++17", "-lineinfo", "--expt-relaxed-constexpr",
    "-Xcompiler", "-fPIC,-O3,-fvisibility=hidden",
    "-I" + str(ROOT / "include"),
    "-Xptxas", "-warn-spills",
]


def nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    return cand


def _headers_mtime() -> float:
    hs = list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + list((ROOT / "include").glob("*.h"))
    return max((h.stat().st_mtime for h in hs), default=0.0)


def _compile(src: Path, obj: Path, verbose: bool) -> tuple[Path, str]:
    cmd = [nvcc()] + NVCC_FLAGS + ["-c", str(src), "-o", str(obj)]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{r.stdout}\n{r.stderr}")
    return obj, r.stdout + r.stderr


def cuda_include() -> Path:
    """Headers of the CUDA toolkit that nvcc() belongs to."""
    return Path(shutil.which(nvcc()) or nvcc()).resolve().parents[1] / "include"


def torch_here() -> tuple[str, str] | None:
    """Version and place of the installed PyTorch, without importing it."""
    spec = importlib.util.find_spec("torch")
    if spec is None or spec.origin is None:
        return None
    return importlib.metadata.version("torch"), spec.origin


def build_torch_ops(force: bool = False) -> Path | None:
    """The CPython module of tensor-level callers; links to libltm_b200.so beside it.
    None, with a message, where there is no PyTorch."""
    found = torch_here()
    if found is None:
        print(f"{OPS.name} is not built: no PyTorch here (the C ABI library does not need it)",
              file=sys.stderr)
        return None
    wanted = "\n".join([*found, sys.version, str(cuda_include())])
    newest = max(p.stat().st_mtime for p in (OPS_SRC, ROOT / "include" / "ltm_b200.h"))
    if (not force and OPS.exists() and OPS.stat().st_mtime >= newest and OPS_FOR.exists()
            and OPS_FOR.read_text() == wanted):
        return OPS
    import sysconfig
    import torch
    from torch.utils import cpp_extension
    inc = cpp_extension.include_paths() + [sysconfig.get_paths()["include"], str(cuda_include())]
    torch_lib = Path(torch.__file__).resolve().parent / "lib"
    tmp = OPS.with_suffix(".so.tmp")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC",
           "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           *[f"-isystem{i}" for i in inc], str(OPS_SRC), "-o", str(tmp), f"-L{LIB.parent}",
           "-l:libltm_b200.so", f"-L{torch_lib}", "-lc10", "-lc10_cuda", "-ltorch_cpu",
           "-ltorch_cuda", "-ltorch_python", "-Wl,-rpath,$ORIGIN", f"-Wl,-rpath,{torch_lib}"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for {OPS_SRC.name}:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, OPS)
    OPS_FOR.parent.mkdir(exist_ok=True)
    OPS_FOR.write_text(wanted)
    return OPS


def build(force: bool = False, jobs: int | None = None, verbose: bool = False) -> Path:
    BUILD.mkdir(exist_ok=True)
    srcs = sorted(CSRC.glob("*.cu"))
    hdr_t = _headers_mtime()
    todo = []
    objs = []
    for s in srcs:
        o = BUILD / (s.stem + ".o")
        objs.append(o)
        if force or not o.exists() or o.stat().st_mtime < max(s.stat().st_mtime, hdr_t):
            todo.append((s, o))
    jobs = jobs or min(len(todo) or 1, os.cpu_count() or 4)
    logs = []
    if todo:
        with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
            for obj, log in ex.map(lambda so: _compile(so[0], so[1], verbose), todo):
                logs.append((obj.name, log))
    if todo or not LIB.exists() or LIB.stat().st_mtime < max(o.stat().st_mtime for o in objs):
        tmp = LIB.with_suffix(".so.tmp")
        cmd = [nvcc()] + ARCH + ["-shared", "-o", str(tmp)] + [str(o) for o in objs] + [
            "-Xcompiler", "-fPIC"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        os.replace(tmp, LIB)
    build_torch_ops(force)
    if verbose:
        for name, log in logs:
            print(f"== {name}\n{log}")
    return LIB


def main() -> int:
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-j", type=int, default=None)
    ap.add_argument("-v", action="store_true", help="print ptxas resource usage")
    a = ap.parse_args()
    print(build(force=a.force, jobs=a.j, verbose=a.v))
    return 0


if __name__ == "__main__":
    sys.exit(main())
